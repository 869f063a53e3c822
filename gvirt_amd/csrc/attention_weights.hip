// What every cached position was attended to: for each sequence, kv head g and position j
//     weights[j][g] (+)= sum over the counted rows r and the heads h of g of  exp(q_rh . k_j) / sum_{j' <= c + r} exp(q_rh . k_j')
// (c cached positions; row r sees positions 0 .. c + r; j <= c + r). Positions of the step itself start at zero, older ones
// keep what earlier steps left. No value of V is involved.
//
// A batch of few rows per sequence (decode steps, short windows) is bound by reading K: the scores are formed once, stored in
// fp32 (a few per cent of the bytes of K) with every row's maximum and sum per chunk of positions, and summed up in a second
// pass over them. A batch of many rows is bound by the exponentials and forms the scores twice instead of storing them (a
// chunk of 2048 rows behind 6144 positions has 0.4 G of them for 28 heads, 1.6 GB in fp32):
//   row statistics: log2 of every row's normaliser. A wave owns 64 M rows (an M row: a counted row and one query head of the
//     kv head) as the columns of S^T = K Q^T, so a row's running maximum and sum live in one lane pair.
//   column sums: a wave owns 64 positions as the columns of S = Q K^T and walks the M rows, so a position's sum lives in one
//     lane pair: no atomics, one owner per weight, the same order of additions in every run.
// Measured, 2 chunks of 2048 rows behind 6144 positions, 28 heads over 4 of 128 elements (210 GFLOP of scores, formed twice): row
// statistics 227-247 us, column sums 258-291 (settled, after a pause), together 0.78-0.87 PFLOP/s (a large bf16 product reaches 1.28):
// the matrix instructions share the SIMDs with 0.8 G exponentials a pass.
#include <algorithm>
#include <type_traits>

#include "attention_common.h"
#include "block_magic.h"
#include "kv8.h"
#include "stage.h"

namespace xlite {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 256;
constexpr uint32_t kRowTile = 4 * 64;         // M rows of a workgroup of the row statistics
constexpr uint32_t kMinSplit = 256;           // positions a split of the row statistics walks at least
// M rows per sequence, on average, up to which the scores are stored: K is read again for every 16 of them and each costs 8 bytes
// a position. 32 sequences of 6000 positions, 8 kv heads of 128, stored / formed twice: 48 rows 334 / 361 us, 64 rows 430 / 342;
// one of 8000: 48 rows 30 / 30; 28 heads over 4: 56 rows 190 / 181. The scratch grows with the limit.
constexpr uint32_t kStoredRows = 32;
// ... and of one sequence: an average says nothing about a chunk beside decode rows. Sequences of more M rows than a tile of the
// row statistics has go through the other kernels, in launches of their own. All stored / long ones apart: 100 decode rows and a
// chunk of 300 rows behind 2000 positions (32 heads over 8) 2340 / 171 us, 300 and a chunk of 1000 (28 over 4) 12060 / 337; 64
// sequences of 1 to 8 rows, none of them long, 159 / 170.
constexpr uint32_t kLongRows = kRowTile;
// Stored scores at a time: kv heads beyond it take turns, and where one head's do not fit they are formed twice. The rows are laid
// out for the widest context that the block tables have room for, whatever the sequences' lengths. (A decode step of 64 sequences
// over tables of 131072 positions: 1028 MB, 196 us; with a limit of 512 MB and so three heads at a time 408.)
constexpr size_t kStoredBytes = 1536ull << 20;

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
    uint32_t block_magic;          // see block_magic()
    float *scores;                 // stored scores: [kv head - head0][M row][pitch], in units of log2
    uint32_t pitch;                // positions of a stored row, a multiple of 64
    uint32_t head0, heads;         // stored scores: the kv heads of a launch
    uint32_t long_rows;            // M rows of a sequence from which on its scores are formed twice (0: those of all, or of none, are)
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

// the n-th sequence whose scores are formed twice, for a whole wave; `batch`: there are fewer
__device__ __forceinline__ uint32_t long_sequence(const WeightsParams &p, uint32_t n, uint32_t lane)
{
    for (uint32_t i0 = 0; i0 < p.batch; i0 += 64) {
        const uint32_t i = i0 + lane;
        uint64_t hits = __ballot(sequence_of(p, min(i, p.batch - 1)).m_rows > p.long_rows && i < p.batch);
        const uint32_t here = static_cast<uint32_t>(__builtin_popcountll(hits));
        if (n < here) {
            for (; n != 0; n--) {
                hits &= hits - 1;
            }
            return i0 + static_cast<uint32_t>(__builtin_ctzll(hits));
        }
        n -= here;
    }
    return p.batch;
}

__device__ __forceinline__ uint64_t slot_of(const WeightsParams &p, const int32_t *table, uint32_t pos)
{
    const uint32_t b = p.block_magic != 0 ? __umulhi(pos, p.block_magic) : pos / p.block_size;
    return static_cast<uint64_t>(static_cast<uint32_t>(table[b])) * p.block_size + (pos - b * p.block_size);
}

// Row tile blockIdx.x of the row statistics, for a whole wave: its sequence and number inside it (which may lie behind its last
// one). False: there is none. The tiles of a sequence are numbered from floor(start * G / TILE) + i (a formula of the prefix sums, at
// least as many ids as it has tiles), or evenly when a window bounds the counted rows; beside stored scores those of the long
// sequences are counted one after the other.
template <uint32_t TILE>
__device__ __forceinline__ bool row_tile_of(const WeightsParams &p, uint32_t lane, uint32_t *seq, uint32_t *mt)
{
    if (p.long_rows != 0) {
        uint32_t left = blockIdx.x;
        for (uint32_t i0 = 0; i0 < p.batch; i0 += 64) {
            const uint32_t rows = sequence_of(p, min(i0 + lane, p.batch - 1)).m_rows;
            const uint32_t tiles = i0 + lane < p.batch && rows > p.long_rows ? ceil_div(rows, TILE) : 0u;
            uint32_t incl = tiles;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t up = __shfl_up(incl, d);
                incl += lane >= static_cast<uint32_t>(d) ? up : 0u;
            }
            const uint64_t behind = __ballot(incl > left);   // the first of these holds the tile
            if (behind != 0) {
                const int at = __builtin_ctzll(behind);
                *seq = i0 + static_cast<uint32_t>(at);
                *mt = left - static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(incl - tiles), at));
                return true;
            }
            left -= static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(incl), 63));
        }
        return false;
    }
    if (p.tiles_per_seq != 0) {
        *seq = blockIdx.x / p.tiles_per_seq;
        *mt = blockIdx.x % p.tiles_per_seq;
        return true;
    }
    auto first_id = [&](uint32_t i) {
        return static_cast<uint32_t>(static_cast<uint64_t>(p.query_start_loc[i]) * p.group / TILE) + i;
    };
    uint32_t at = 0, hi = p.batch;
    while (hi - at > 1) {
        const uint32_t mid = (at + hi) >> 1;
        if (first_id(mid) <= blockIdx.x) {
            at = mid;
        } else {
            hi = mid;
        }
    }
    *seq = at;
    *mt = blockIdx.x - first_id(at);
    return true;
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

// tiles of 32 rows of a wave (head_dim 256: the registers hold one), positions of a staged tile
template <int D>
constexpr int kRowTiles = D == 256 ? 1 : 2;
template <int D>
constexpr int kStagedPositions = D == 256 ? 32 : 64;

template <typename T, int D, int KVF>
__global__ void __launch_bounds__(kThreads)
row_stats_kernel(const WeightsParams p)
{
    constexpr int KS = D / 16;
    constexpr int RT = kRowTiles<D>;
    constexpr bool KV8 = KVF != XLITE_HIP_KV_SAME;
    constexpr uint32_t ROWB = D * (KV8 ? 1 : 2);
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, half = lane >> 5;
    const uint32_t kvh = blockIdx.z, split = blockIdx.y, G = p.group;
    constexpr uint32_t TILE = 4 * 32 * RT;

    uint32_t seq, mt;
    if (!row_tile_of<TILE>(p, lane, &seq, &mt)) {
        return;
    }
    const Sequence s = sequence_of(p, seq);
    const uint32_t m_wave = mt * TILE + wave * 32 * RT;
    if (m_wave >= s.m_rows) {
        return;
    }
    uint32_t vis[RT];                                                            // of this lane's rows
    const uint32_t vis_first = s.cached + s.first + m_wave / G + 1;              // of the wave's first row, the least
    const uint32_t vis_last = s.cached + s.first + min(m_wave + 32 * RT - 1, s.m_rows - 1) / G + 1;
    const uint32_t begin = split * p.split_len, end = min(vis_last, begin + p.split_len);
    const int32_t *table = p.block_tables + static_cast<uint64_t>(seq) * p.max_num_block;

    float m_run[RT], l_run[RT];
    uint4 qreg[RT][KS];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const uint32_t m = min(m_wave + rt * 32 + col, s.m_rows - 1);
        const uint32_t r = s.first + m / G;
        vis[rt] = s.cached + r + 1;
        m_run[rt] = -INFINITY;
        l_run[rt] = 0.f;
        const uint16_t *src = p.q + static_cast<uint64_t>(s.start + r) * p.q_tok_stride + static_cast<uint64_t>(kvh * G + m % G) * D;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            qreg[rt][ks] = *reinterpret_cast<const uint4 *>(src + ks * 16 + half * 8);
        }
    }
    if (begin < end) {
        // a tile's K chunks are requested one tile ahead, its block-table entries two (positions past the end repeat the
        // last one; their scores are masked)
        typedef typename std::conditional<KV8, uint2, uint4>::type raw_t;
        raw_t next[KS];
        float scale_next = 1.f;
        auto slot_ahead = [&](uint32_t t0) __attribute__((always_inline)) { return slot_of(p, table, min(t0 + col, end - 1)) * p.n_kv_heads + kvh; };
        auto request = [&](uint64_t at) __attribute__((always_inline)) {
            const unsigned char *row = p.k_cache + at * ROWB;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                next[ks] = *reinterpret_cast<const raw_t *>(row + (2 * ks + half) * sizeof(raw_t));
            }
            if constexpr (KV8) {
                scale_next = p.k_scale[at];
            }
        };
        request(slot_ahead(begin));
        uint64_t at_next = slot_ahead(begin + 32);
        for (uint32_t t0 = begin; t0 < end; t0 += 32) {
            uint4 kop[KS];
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                if constexpr (KV8) {
                    kop[ks] = dequant8<T, KVF>(next[ks], 1.0f);
                } else {
                    kop[ks] = next[ks];
                }
            }
            const float scale = scale_next;
            request(at_next);
            at_next = slot_ahead(t0 + 64);
            f32x16_t S[RT];
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    S[rt][k] = 0.f;
                }
            }
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    S[rt] = mfma32<T>(kop[ks], qreg[rt][ks], S[rt]);
                }
            }
            const bool masked = t0 + 32 > min(vis_first, end);
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                if constexpr (KV8) {   // the scale of position t0 + col; register k holds another one
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        S[rt][k] *= __shfl(scale, static_cast<int>((k / 4) * 8 + half * 4 + (k % 4)));
                    }
                }
                if (masked) {
                    const uint32_t lim = min(vis[rt], end);
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        S[rt][k] = t0 + (k / 4) * 8 + half * 4 + (k % 4) < lim ? S[rt][k] : -INFINITY;
                    }
                }
                float mx = m_run[rt];
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    mx = fmaxf(mx, S[rt][k]);
                }
                const float m_safe = mx == -INFINITY ? 0.f : mx;
                const float neg = -m_safe * kLog2e;
                float sum = 0.f;
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    sum += fast_exp2(__builtin_fmaf(S[rt][k], kLog2e, neg));
                }
                l_run[rt] = l_run[rt] * fast_exp2((m_run[rt] - m_safe) * kLog2e) + sum;
                m_run[rt] = mx;
            }
        }
    }
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        // the two halves of a row's positions
        const float m_other = __shfl_xor(m_run[rt], 32), l_other = __shfl_xor(l_run[rt], 32);
        const float m_all = fmaxf(m_run[rt], m_other);
        const float m_safe = m_all == -INFINITY ? 0.f : m_all;
        const float l_all = l_run[rt] * fast_exp2((m_run[rt] - m_safe) * kLog2e) + l_other * fast_exp2((m_other - m_safe) * kLog2e);
        const uint32_t m = m_wave + rt * 32 + col;
        if (half == 0 && m < s.m_rows) {
            const uint64_t i = static_cast<uint64_t>(kvh) * p.m_total + static_cast<uint64_t>(s.start + s.first) * G + m;
            if (p.splits == 1) {
                p.norm[i] = -(m_all * kLog2e + __log2f(l_all));
            } else {
                *reinterpret_cast<float2 *>(p.stats + (static_cast<uint64_t>(split) * p.n_kv_heads * p.m_total + i) * 2) =
                    make_float2(m_all * kLog2e, l_all);
            }
        }
    }
}

// The same for 16-bit caches, K tiles of 64 positions (32 of head_dim 256) copied straight into LDS (a ring of three) and
// shared by the four waves. Read from memory by every wave, as above, a K chunk of 32 positions touches 32 lines per
// instruction and every line four times: the vector cache's look-ups took longer than the products and the exponentials.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2)
row_stats_staged_kernel(const WeightsParams p)
{
    constexpr int KS = D / 16, RT = kRowTiles<D>, BN = kStagedPositions<D>, STAGES = 3;
    constexpr uint32_t ROWB = D * 2, STAGE = BN * ROWB, TILE = 4 * 32 * RT;
    constexpr int PPC = 1024 / ROWB;           // positions per copy
    constexpr int CPW = BN / PPC / 4;          // copies per wave and tile
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    uint32_t *tbl = reinterpret_cast<uint32_t *>(smem + STAGES * STAGE);
    const uint32_t smem_addr = stage::lds_address(smem);
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
    const uint32_t kvh = blockIdx.z, split = blockIdx.y, G = p.group;
    uint32_t seq, mt;
    if (!row_tile_of<TILE>(p, lane, &seq, &mt)) {
        return;
    }
    const Sequence s = sequence_of(p, seq);
    const uint32_t m_first = mt * TILE;
    if (m_first >= s.m_rows) {
        return;
    }
    const uint32_t m_wave = min(m_first + wave * 32 * RT, s.m_rows - 1);         // (a wave without rows repeats the last one)
    uint32_t vis[RT];
    const uint32_t vis_first = s.cached + s.first + m_wave / G + 1;
    // the workgroup's range: what its last row sees
    const uint32_t vis_last = s.cached + s.first + min(m_first + TILE - 1, s.m_rows - 1) / G + 1;
    const uint32_t begin = split * p.split_len, end = min(vis_last, begin + p.split_len);
    const int32_t *table = p.block_tables + static_cast<uint64_t>(seq) * p.max_num_block;
    float m_run[RT], l_run[RT];
    uint4 qreg[RT][KS];
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const uint32_t m = min(m_wave + rt * 32 + col, s.m_rows - 1);
        const uint32_t r = s.first + m / G;
        vis[rt] = s.cached + r + 1;
        m_run[rt] = -INFINITY;
        l_run[rt] = 0.f;
        const uint16_t *src = p.q + static_cast<uint64_t>(s.start + r) * p.q_tok_stride + static_cast<uint64_t>(kvh * G + m % G) * D;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            qreg[rt][ks] = *reinterpret_cast<const uint4 *>(src + ks * 16 + half * 8);
        }
    }
    if (begin < end) {
        const uint32_t blk0 = begin / p.block_size, blk1 = (end - 1) / p.block_size;
        for (uint32_t i = threadIdx.x; i <= blk1 - blk0; i += kThreads) {
            tbl[i] = static_cast<uint32_t>(table[blk0 + i]);
        }
        // complete these loads before any copy is issued
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                asm volatile("" : "+v"(qreg[rt][ks].x), "+v"(qreg[rt][ks].y), "+v"(qreg[rt][ks].z), "+v"(qreg[rt][ks].w));
            }
        }
        __syncthreads();
        const uint32_t pitch = p.n_kv_heads * ROWB;
        uint32_t c_row[CPW], c_off[CPW];
#pragma unroll
        for (int i = 0; i < CPW; i++) {
            uint32_t chunk;
            stage::copy_source<D>(lane, PPC * (CPW * wave + i), &c_row[i], &chunk);
            c_off[i] = chunk << 4;
        }
        // copies of tile `tile` of the range into stage tile % 3; the positions of a copy share a block, those past the end
        // repeat the last one (their scores are masked)
        auto issue = [&](uint32_t tile) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < CPW; i++) {
                const uint32_t pos = PPC * (CPW * wave + i);
                const uint32_t t_raw = begin + tile * BN + pos, lim = end - 1;
                const uint32_t t = min(t_raw, lim) & ~static_cast<uint32_t>(PPC - 1);
                const uint32_t rel = min(t_raw + c_row[i], lim) - t;
                const uint32_t blk = __umulhi(t, p.block_magic);
                const uint32_t phys = __builtin_amdgcn_readfirstlane(tbl[blk - blk0]);
                const uint64_t row0 = static_cast<uint64_t>(phys) * p.block_size + (t - blk * p.block_size);
                const char *kb = reinterpret_cast<const char *>(p.k_cache) + row0 * pitch + kvh * ROWB;
                stage::copy_1k(smem_addr + (tile % STAGES) * STAGE + pos * ROWB, rel * pitch + c_off[i], kb);
            }
        };
        const uint32_t n_tiles = ceil_div(end - begin, static_cast<uint32_t>(BN));
        const uint32_t row_off = stage::row_offset<D>(col), x = stage::row_swizzle<D>(col, half);
        issue(0);
        issue(1);
        for (uint32_t tile = 0; tile < n_tiles; tile++) {
            stage::wait<CPW>();   // this wave's share of `tile` has landed
            __syncthreads();      // ... and everybody else's; stage (tile - 1) % 3 is free
            issue(tile + 2);
#pragma unroll
            for (int h = 0; h < BN / 32; h++) {
                const uint32_t t0 = begin + tile * BN + h * 32;
                const unsigned char *base = smem + (tile % STAGES) * STAGE + h * 32 * ROWB + row_off;
                uint4 kop[KS];
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    kop[ks] = *reinterpret_cast<const uint4 *>(base + stage::chunk_offset(ks, x));
                }
                f32x16_t S[RT];
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        S[rt][k] = 0.f;
                    }
                }
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
#pragma unroll
                    for (int rt = 0; rt < RT; rt++) {
                        S[rt] = mfma32<T>(kop[ks], qreg[rt][ks], S[rt]);
                    }
                }
                const bool masked = t0 + 32 > min(vis_first, end);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    if (masked) {
                        const uint32_t lim = min(vis[rt], end);
#pragma unroll
                        for (int k = 0; k < 16; k++) {
                            S[rt][k] = t0 + (k / 4) * 8 + half * 4 + (k % 4) < lim ? S[rt][k] : -INFINITY;
                        }
                    }
                    // The reference of a row's exponentials moves only when a tile's sum says so (the first tile's does): any
                    // reference within 2^60 of the maximum gives the same sum in fp32, and finding every tile's maximum is
                    // a tenth of the kernel's vector instructions.
                    float sum = 0.f;
                    const float neg = -m_run[rt] * kLog2e;
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        sum += fast_exp2(__builtin_fmaf(S[rt][k], kLog2e, neg));
                    }
                    if (__any(!(sum < 0x1p60f))) {   // (the first tile: the reference is -infinity, the sum infinite or NaN)
                        float mx = m_run[rt];
#pragma unroll
                        for (int k = 0; k < 16; k++) {
                            mx = fmaxf(mx, S[rt][k]);
                        }
                        const float m_safe = mx == -INFINITY ? 0.f : mx;
                        sum = 0.f;
#pragma unroll
                        for (int k = 0; k < 16; k++) {
                            sum += fast_exp2(__builtin_fmaf(S[rt][k], kLog2e, -m_safe * kLog2e));
                        }
                        l_run[rt] *= fast_exp2((m_run[rt] - m_safe) * kLog2e);
                        m_run[rt] = mx;
                    }
                    l_run[rt] += sum;
                }
            }
        }
        stage::wait<0>();   // (nothing is left on its way into LDS when the workgroup ends)
    }
#pragma unroll
    for (int rt = 0; rt < RT; rt++) {
        const float m_other = __shfl_xor(m_run[rt], 32), l_other = __shfl_xor(l_run[rt], 32);
        const float m_all = fmaxf(m_run[rt], m_other);
        const float m_safe = m_all == -INFINITY ? 0.f : m_all;
        const float l_all = l_run[rt] * fast_exp2((m_run[rt] - m_safe) * kLog2e) + l_other * fast_exp2((m_other - m_safe) * kLog2e);
        const uint32_t m = m_first + wave * 32 * RT + rt * 32 + col;
        if (half == 0 && m < s.m_rows) {
            const uint64_t i = static_cast<uint64_t>(kvh) * p.m_total + static_cast<uint64_t>(s.start + s.first) * G + m;
            if (p.splits == 1) {
                p.norm[i] = -(m_all * kLog2e + __log2f(l_all));
            } else {
                *reinterpret_cast<float2 *>(p.stats + (static_cast<uint64_t>(split) * p.n_kv_heads * p.m_total + i) * 2) =
                    make_float2(m_all * kLog2e, l_all);
            }
        }
    }
}

// joins the splits of every row (rows that nobody counted hold whatever the workspace held; nobody reads them): L lanes a row,
// each every L-th split, so that one row of a long context (hundreds of splits) is not one chain of loads
template <int L>
__global__ void __launch_bounds__(256)
join_stats_kernel(const float *__restrict__ stats, float *__restrict__ norm, uint32_t rows, uint32_t splits)
{
    const uint64_t at = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
    const uint32_t i = static_cast<uint32_t>(min(at / L, static_cast<uint64_t>(rows - 1))), part = threadIdx.x % L;
    float m = -INFINITY, l = 0.f;
    for (uint32_t s = part; s < splits; s += L) {
        const float2 x = *reinterpret_cast<const float2 *>(stats + (static_cast<uint64_t>(s) * rows + i) * 2);
        const float mx = fmaxf(m, x.x), safe = mx == -INFINITY ? 0.f : mx;
        l = l * fast_exp2(m - safe) + x.y * fast_exp2(x.x - safe);
        m = mx;
    }
#pragma unroll
    for (int d = 1; d < L; d <<= 1) {
        const float m_other = __shfl_xor(m, d), l_other = __shfl_xor(l, d);
        const float mx = fmaxf(m, m_other), safe = mx == -INFINITY ? 0.f : mx;
        l = l * fast_exp2(m - safe) + l_other * fast_exp2(m_other - safe);
        m = mx;
    }
    if (part == 0 && at / L < rows) {
        norm[i] = -(m + __log2f(l));
    }
}

// Query rows copied straight into LDS, 32 M rows for each turn (four waves, 64 positions each, 32 of head_dim 256) at a time, and
// their normalisers with them. As many turns as the registers hold waves: the exponentials of
// a tile (96 vector instructions, 300 cycles with four waves on a SIMD, 410 with one) run beside the products of the others.
template <int D>
constexpr int kTurns = D == 256 ? 2 : D == 128 ? 3 : 4;
template <int D>
constexpr int kColumnTiles = D == 256 ? 1 : 2;   // tiles of 32 positions of a wave

template <typename T, int D, int KVF>
__global__ void __launch_bounds__(kTurns<D> * kThreads)
column_sums_kernel(const WeightsParams p)
{
    constexpr int KS = D / 16, PT = kColumnTiles<D>, STAGES = 3, TURNS = kTurns<D>, ROWS = 32 * TURNS;
    constexpr uint32_t ROWB = D * (KVF == XLITE_HIP_KV_SAME ? 2 : 1), QROWB = D * 2;
    constexpr uint32_t QBYTES = ROWS * QROWB, STAGE = QBYTES + 4 * TURNS * 256;   // the rows, then each wave's normalisers
    constexpr int RPC = 1024 / QROWB, CPW = 8 / RPC;                    // rows per copy, copies per wave
    constexpr uint32_t WG = 4 * 32 * PT;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    __shared__ float other[TURNS][4][32 * PT];
    const uint32_t smem_addr = stage::lds_address(smem);
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
    const uint32_t kvh = blockIdx.z, G = p.group;
    const uint32_t seq = p.long_rows == 0 ? blockIdx.y : long_sequence(p, blockIdx.y, lane);
    if (seq >= p.batch) {
        return;
    }
    const uint32_t mine = wave & 3u, turn = wave >> 2;   // which 64 positions, and which 32 of the staged rows
    const Sequence s = sequence_of(p, seq);
    const uint32_t total = s.cached + s.nodes;
    const uint32_t wg0 = blockIdx.x * WG;
    if (s.nodes == 0 || wg0 >= total) {
        return;
    }
    const uint32_t p0 = wg0 + mine * 32 * PT;   // the wave's first position
    const int32_t *table = p.block_tables + static_cast<uint64_t>(seq) * p.max_num_block;
    uint64_t at[PT];
    uint4 kreg[PT][KS];
    float mul[PT], acc[PT];
#pragma unroll
    for (int pt = 0; pt < PT; pt++) {
        at[pt] = slot_of(p, table, min(p0 + pt * 32 + col, total - 1)) * p.n_kv_heads + kvh;
        const unsigned char *row = p.k_cache + at[pt] * ROWB;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            kreg[pt][ks] = cache_chunk<T, KVF>(row, 2 * ks + half);
        }
        mul[pt] = kLog2e;
        acc[pt] = 0.f;
        if constexpr (KVF != XLITE_HIP_KV_SAME) {
            mul[pt] *= p.k_scale[at[pt]];
        }
    }
    // complete these loads before any copy is issued
#pragma unroll
    for (int pt = 0; pt < PT; pt++) {
        asm volatile("" : "+v"(mul[pt]));
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            asm volatile("" : "+v"(kreg[pt][ks].x), "+v"(kreg[pt][ks].y), "+v"(kreg[pt][ks].z), "+v"(kreg[pt][ks].w));
        }
    }
    // from the first row that sees the workgroup's first position on (rows before it see none of its positions)
    const uint32_t m_begin = (wg0 > s.cached + s.first ? (wg0 - s.cached - s.first) * G : 0u) & ~31u;
    const uint32_t rows = s.m_rows - m_begin, n_it = ceil_div(rows, static_cast<uint32_t>(ROWS));   // (the last row sees every position: rows > 0)
    const uint64_t tok0 = s.start + s.first;
    const float *norm = p.norm + static_cast<uint64_t>(kvh) * p.m_total + tok0 * G + m_begin;
    const uint16_t *q0 = p.q + tok0 * p.q_tok_stride + static_cast<uint64_t>(kvh * G) * D;
    // a lane's rows of the copies: M row m_begin + ROWS it + c_m, as (token, head); rows past the end repeat the last one
    uint32_t c_m[CPW], c_r[CPW], c_h[CPW], c_chunk[CPW];
#pragma unroll
    for (int i = 0; i < CPW; i++) {
        const uint32_t first = RPC * (CPW * wave + i);
        uint32_t row;
        stage::copy_source<D>(lane, first, &row, &c_chunk[i]);
        c_m[i] = first + row;
        c_r[i] = (m_begin + c_m[i]) / G;
        c_h[i] = (m_begin + c_m[i]) - c_r[i] * G;
    }
    const uint32_t dr = ROWS / G, dh = ROWS - dr * G, r_last = (s.m_rows - 1) / G;
    uint32_t m_ahead = 0;   // M rows (from m_begin) that the next copies start at
    auto issue = [&](uint32_t slot) __attribute__((always_inline)) {
        const uint32_t st = smem_addr + slot * STAGE;
#pragma unroll
        for (int i = 0; i < CPW; i++) {
            const bool in = m_ahead + c_m[i] < rows;
            const uint32_t r = in ? c_r[i] : r_last, h = in ? c_h[i] : G - 1;
            stage::copy_lanes_16(st + RPC * (CPW * wave + i) * QROWB, q0 + static_cast<uint64_t>(r) * p.q_tok_stride + h * D + c_chunk[i] * 8);
            c_h[i] += dh;
            c_r[i] += dr;
            const bool over = c_h[i] >= G;
            c_h[i] -= over ? G : 0u;
            c_r[i] += over ? 1u : 0u;
        }
        stage::copy_lanes_4(st + QBYTES + wave * 256, norm + min(m_ahead + 32 * turn + (lane & 31u), rows - 1));
        m_ahead += ROWS;
    };
    const uint32_t row_off = stage::row_offset<D>(col), x = stage::row_swizzle<D>(col, half);
    uint32_t slot = 0;
    issue(0);
    issue(1);
    for (uint32_t it = 0; it < n_it; it++) {
        stage::wait<CPW + 1>();   // this wave's share of the stage has landed
        __syncthreads();          // ... and everybody else's; the stage before it is free
        issue(slot == 0 ? 2u : slot - 1);
        const unsigned char *st = smem + slot * STAGE;
        slot = slot == 2 ? 0u : slot + 1;
        const uint32_t m0 = m_begin + it * ROWS + turn * 32;
        // (a tile of rows that see none of the wave's positions, and one past the end)
        if (m0 >= s.m_rows || s.cached + s.first + (m0 + 31) / G < p0) {
            continue;
        }
        uint4 qop[KS];
        const unsigned char *base = st + turn * 32 * QROWB + row_off;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            qop[ks] = *reinterpret_cast<const uint4 *>(base + stage::chunk_offset(ks, x));
        }
        float n[16];
        const float *nl = reinterpret_cast<const float *>(st + QBYTES + wave * 256) + half * 4;
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const float4 v = *reinterpret_cast<const float4 *>(nl + g * 8);
            n[4 * g] = v.x;
            n[4 * g + 1] = v.y;
            n[4 * g + 2] = v.z;
            n[4 * g + 3] = v.w;
        }
        f32x16_t S[PT];
#pragma unroll
        for (int pt = 0; pt < PT; pt++) {
#pragma unroll
            for (int k = 0; k < 16; k++) {
                S[pt][k] = 0.f;
            }
        }
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
#pragma unroll
            for (int pt = 0; pt < PT; pt++) {
                S[pt] = mfma32<T>(qop[ks], kreg[pt][ks], S[pt]);
            }
        }
        const bool masked = m0 + 32 > s.m_rows || p0 + 32 * PT - 1 > s.cached + s.first + m0 / G;
#pragma unroll
        for (int pt = 0; pt < PT; pt++) {
            float sum = 0.f;
            if (masked) {
                // of the lane's rows, those from the first one that sees the position on
                const uint32_t t = p0 + pt * 32 + col;
                const uint32_t from = t > s.cached + s.first ? (t - s.cached - s.first) * G : 0u;
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    const uint32_t mk = m0 + (k / 4) * 8 + half * 4 + (k % 4);
                    const float e = fast_exp2(__builtin_fmaf(S[pt][k], mul[pt], n[k]));
                    sum += mk < s.m_rows && mk >= from ? e : 0.f;
                }
            } else {
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    sum += fast_exp2(__builtin_fmaf(S[pt][k], mul[pt], n[k]));
                }
            }
            acc[pt] += sum;   // (a tile's sum first: 16 additions, then one per tile, not one chain over every row)
        }
    }
    stage::wait<0>();
#pragma unroll
    for (int pt = 0; pt < PT; pt++) {
        acc[pt] += __shfl_xor(acc[pt], 32);
        if (turn != 0 && half == 0) {
            other[turn][mine][pt * 32 + col] = acc[pt];
        }
    }
    __syncthreads();
    if (turn == 0 && half == 0) {
#pragma unroll
        for (int pt = 0; pt < PT; pt++) {
            const uint32_t t = p0 + pt * 32 + col;
            if (t < total) {
                float sum = acc[pt];
#pragma unroll
                for (int u = 1; u < TURNS; u++) {
                    sum += other[u][mine][pt * 32 + col];
                }
                p.weights[at[pt]] = t < s.cached ? p.weights[at[pt]] + sum : sum;
            }
        }
    }
}

// ---- few rows: scores stored ------------------------------------------------------------------------------------------------
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4v_t;
template <typename T>
__device__ __forceinline__ f32x4v_t mfma16(const uint4 &a, const uint4 &b, f32x4v_t c)
{
    if constexpr (T::kCode == XLITE_HIP_BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    }
}

// where a sequence's stored rows begin (in M rows of a kv head): window rows per sequence, or its tokens
__device__ __forceinline__ uint32_t stored_base(const WeightsParams &p, uint32_t seq, const Sequence &s)
{
    return (p.window != 0 ? seq * p.window : s.start) * p.group;
}

// A wave takes the positions of one kv head, of a chunk [chunk * split_len, + split_len): K rows are copied as they stand into
// the wave's own ring of stages in LDS (no barriers), a whole row by neighbouring lanes, 16 rows are the A operand of a
// product with 16 M rows as columns. It leaves the scores and every row's maximum and sum over the chunk. Waves of a
// workgroup: kv heads side by side, and where there are fewer than four, neighbouring chunks.
// Bound by memory. Measured, 64 decode rows of 8 kv heads over up to 4096 positions of 128 elements (340 MB of K): 73 us, 4.7
// TB/s; 79 without the hint that nobody reads the bytes again, 89 with the operand read straight from memory (a row in four
// requests of 64 bytes). A ring of four stages (two workgroups a compute unit instead of three) is no faster.
template <int D, bool KV8>
struct StoredTile {
    static constexpr uint32_t ROWB = D * (KV8 ? 1 : 2);
    static constexpr uint32_t C = ROWB / 16;                                    // 16-byte chunks of a row
    static constexpr uint32_t BN = ROWB * 16 > 4096 ? 16 : 4096 / ROWB;         // positions of a stage: 16 .. 64
    static constexpr uint32_t BYTES = BN * ROWB, COPIES = BYTES / 1024;
    static constexpr uint32_t SCALES = KV8 ? 256 : 0;                           // a stage's K scales, behind its rows
    static constexpr int STAGES = D == 256 ? 2 : 3;
    static constexpr uint32_t RING = STAGES * (BYTES + SCALES);
    // 16-byte chunk i of a stage, exchanged within its 256 bytes: 16 rows' chunks of one column lie in different banks
    static __device__ __forceinline__ uint32_t exchanged(uint32_t i)
    {
        return i ^ ((C == 32 ? i >> 5 : i >> 4) & 15u);
    }
};
constexpr uint32_t kStoredWaves = 4;

__host__ __device__ __forceinline__ uint32_t stored_table(uint32_t split_len, uint32_t block_size)   // entries, in whole 16 bytes
{
    return (split_len / block_size + 2 + 3) / 4 * 4;
}

template <typename T, int D, int KVF>
__global__ void __launch_bounds__(64 * kStoredWaves)
store_scores_kernel(const WeightsParams p)
{
    constexpr bool KV8 = KVF != XLITE_HIP_KV_SAME;
    typedef StoredTile<D, KV8> Tile;
    constexpr int KS = D / 32, NT = Tile::BN / 16, S = Tile::STAGES, C = Tile::C;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, jq = lane >> 4;
    const uint32_t heads = min(p.heads, kStoredWaves), per_wg = kStoredWaves / heads;   // kv heads and chunks of a workgroup
    const uint32_t parts = ceil_div(p.heads, heads);
    const uint32_t local = blockIdx.x % parts * heads + wave % heads, chunk = blockIdx.x / parts * per_wg + wave / heads;
    const uint32_t kvh = p.head0 + local;
    const uint32_t seq = blockIdx.y, G = p.group;
    const Sequence s = sequence_of(p, seq);
    const uint32_t total = s.cached + s.nodes;
    const uint32_t begin = chunk * p.split_len, end = min(total, begin + p.split_len);
    if (wave >= heads * per_wg || local >= p.heads || s.nodes == 0 || chunk >= p.splits || (p.long_rows != 0 && s.m_rows > p.long_rows)) {
        return;
    }
    const uint32_t entries = stored_table(p.split_len, p.block_size);
    unsigned char *ring = smem + wave * (Tile::RING + entries * 4);
    uint32_t *tbl = reinterpret_cast<uint32_t *>(ring + Tile::RING);
    const uint32_t ring_addr = stage::lds_address(smem) + wave * (Tile::RING + entries * 4);
    const uint32_t base = stored_base(p, seq, s);
    const uint64_t rows0 = static_cast<uint64_t>(local) * p.m_total + base;
    auto block_of = [&](uint32_t pos) __attribute__((always_inline)) { return p.block_magic != 0 ? __umulhi(pos, p.block_magic) : pos / p.block_size; };
    const uint32_t blk0 = block_of(begin);
    if (begin < end) {
        const int32_t *table = p.block_tables + static_cast<uint64_t>(seq) * p.max_num_block + blk0;
        const uint32_t blocks = block_of(end - 1) - blk0 + 1;
        for (uint32_t i = lane; i < blocks; i += 64) {
            tbl[i] = static_cast<uint32_t>(table[i]);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    // row of K, of a scale
    auto row_at = [&](uint32_t pos) __attribute__((always_inline)) {
        const uint32_t t = min(pos, end - 1), b = block_of(t);
        return (static_cast<uint64_t>(tbl[b - blk0]) * p.block_size + (t - b * p.block_size)) * p.n_kv_heads + kvh;
    };
    // copies of the chunk's tile `it` into stage `slot` (positions past the end repeat the last one: their scores are masked, and
    // every tile is the same number of copies)
    auto issue = [&](uint32_t it, uint32_t slot, bool once) __attribute__((always_inline)) {
        const uint32_t t0 = begin + it * Tile::BN, st = ring_addr + slot * (Tile::BYTES + Tile::SCALES);
#pragma unroll
        for (uint32_t i = 0; i < Tile::COPIES; i++) {
            const uint32_t x = Tile::exchanged(64 * i + lane);
            const unsigned char *src = p.k_cache + row_at(t0 + x / C) * Tile::ROWB + x % C * 16;
            if (once) {
                stage::copy_lanes_16_once(st + i * 1024, src);
            } else {
                stage::copy_lanes_16(st + i * 1024, src);
            }
        }
        if constexpr (KV8) {
            stage::copy_lanes_4(st + Tile::BYTES, p.k_scale + row_at(t0 + min(lane, Tile::BN - 1)));
        }
    };
    for (uint32_t m0 = 0; m0 < s.m_rows; m0 += 16) {
        const uint32_t m = min(m0 + col, s.m_rows - 1);
        const uint32_t r = s.first + m / G;
        const uint32_t lim = s.cached + r + 1;
        const bool once = m0 + 16 >= s.m_rows;   // no further rows read the chunk again
        float m_run = -INFINITY, l_run = 0.f;
        if (begin < end) {
            const uint16_t *src = p.q + static_cast<uint64_t>(s.start + r) * p.q_tok_stride + static_cast<uint64_t>(kvh * G + m % G) * D;
            uint4 qreg[KS];
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                qreg[ks] = *reinterpret_cast<const uint4 *>(src + ks * 32 + jq * 8);
            }
            // complete these loads before any copy is issued
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                asm volatile("" : "+v"(qreg[ks].x), "+v"(qreg[ks].y), "+v"(qreg[ks].z), "+v"(qreg[ks].w));
            }
            float *out = p.scores + (rows0 + m0 + col) * p.pitch;
            const uint32_t n_it = ceil_div(end - begin, Tile::BN);
#pragma unroll
            for (int i = 0; i < S - 1; i++) {
                issue(i, i, once);
            }
            uint32_t slot = 0;
            for (uint32_t it = 0; it < n_it; it++) {
                stage::wait<(S - 2) * (Tile::COPIES + (KV8 ? 1 : 0))>();   // this tile has landed (the scores' stores make it wait for a little more)
                issue(it + S - 1, slot == 0 ? S - 1 : slot - 1, once);    // into the stage that the last iteration has read
                const unsigned char *st = ring + slot * (Tile::BYTES + Tile::SCALES);
                slot = slot == S - 1 ? 0u : slot + 1;
                const uint32_t t0 = begin + it * Tile::BN;
                f32x4v_t sc[NT];
                float mx = m_run;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    sc[nt] = f32x4v_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int ks = 0; ks < KS; ks++) {
                        if constexpr (KV8) {
                            const uint32_t at = Tile::exchanged((nt * 16 + col) * C + 2 * ks + (jq >> 1)) * 16 + (jq & 1u) * 8;
                            sc[nt] = mfma16<T>(dequant8<T, KVF>(*reinterpret_cast<const uint2 *>(st + at), 1.0f), qreg[ks], sc[nt]);
                        } else {
                            const uint32_t at = Tile::exchanged((nt * 16 + col) * C + 4 * ks + jq) * 16;
                            sc[nt] = mfma16<T>(*reinterpret_cast<const uint4 *>(st + at), qreg[ks], sc[nt]);
                        }
                    }
                    f32x4v_t mul = {kLog2e, kLog2e, kLog2e, kLog2e};
                    if constexpr (KV8) {
                        mul *= *reinterpret_cast<const f32x4v_t *>(st + Tile::BYTES + (nt * 16 + 4 * jq) * 4);
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        sc[nt][e] *= mul[e];
                        mx = fmaxf(mx, t0 + nt * 16 + 4 * jq + e < lim ? sc[nt][e] : -INFINITY);
                    }
                    if (m0 + col < s.m_rows) {   // (positions past the end: inside the row's pitch, nobody reads them)
                        *reinterpret_cast<float4 *>(out + t0 + nt * 16 + 4 * jq) = make_float4(sc[nt][0], sc[nt][1], sc[nt][2], sc[nt][3]);
                    }
                }
                const float m_safe = mx == -INFINITY ? 0.f : mx;
                float sum = 0.f;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float x = fast_exp2(sc[nt][e] - m_safe);
                        sum += t0 + nt * 16 + 4 * jq + e < lim ? x : 0.f;
                    }
                }
                l_run = l_run * fast_exp2(m_run - m_safe) + sum;
                m_run = mx;
            }
            stage::wait<0>();   // (nothing is left on its way into LDS)
        }
        // the row's four lanes
#pragma unroll
        for (int d = 16; d <= 32; d <<= 1) {
            const float m_other = __shfl_xor(m_run, d), l_other = __shfl_xor(l_run, d);
            const float m_all = fmaxf(m_run, m_other);
            const float m_safe = m_all == -INFINITY ? 0.f : m_all;
            l_run = l_run * fast_exp2(m_run - m_safe) + l_other * fast_exp2(m_other - m_safe);
            m_run = m_all;
        }
        if (jq == 0 && m0 + col < s.m_rows) {
            *reinterpret_cast<float2 *>(p.stats + (static_cast<uint64_t>(chunk) * p.heads * p.m_total + rows0 + m0 + col) * 2) =
                make_float2(m_run, l_run);
        }
    }
}

// a thread per position: the stored scores of its kv heads' rows
__global__ void __launch_bounds__(kThreads)
sum_scores_kernel(const WeightsParams p)
{
    const uint32_t seq = blockIdx.y, G = p.group;
    const Sequence s = sequence_of(p, seq);
    const uint32_t total = s.cached + s.nodes, t = blockIdx.x * kThreads + threadIdx.x;
    if (s.nodes == 0 || t >= total || (p.long_rows != 0 && s.m_rows > p.long_rows)) {
        return;
    }
    const int32_t *table = p.block_tables + static_cast<uint64_t>(seq) * p.max_num_block;
    float *w = p.weights + slot_of(p, table, t) * p.n_kv_heads + p.head0;
    const uint32_t base = stored_base(p, seq, s);
    // rows that see the position: from the first counted row r with s.cached + r >= t on
    const uint32_t m_first = t > s.cached + s.first ? (t - s.cached - s.first) * G : 0u;
    for (uint32_t kvh = blockIdx.z; kvh < p.heads; kvh += gridDim.z) {   // (from head0 on)
        const uint64_t rows0 = static_cast<uint64_t>(kvh) * p.m_total + base;
        const float *norm = p.norm + rows0;
        const float *score = p.scores + rows0 * p.pitch + t;
        const float old = w[kvh];
        float acc = 0.f;
        for (uint32_t m0 = 0; m0 < s.m_rows; m0 += 8) {
            float x[8];
#pragma unroll
            for (int u = 0; u < 8; u++) {
                x[u] = score[static_cast<uint64_t>(min(m0 + u, s.m_rows - 1)) * p.pitch];
            }
            float sum = 0.f;
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const float e = fast_exp2(x[u] + norm[min(m0 + u, s.m_rows - 1)]);
                sum += m0 + u >= m_first && m0 + u < s.m_rows ? e : 0.f;
            }
            acc += sum;
        }
        w[kvh] = t < s.cached ? old + acc : acc;
    }
}

// ---- the plan of a call: which kernels, how many pieces, how much scratch -----------------------------------------------------
// Scores stored (`heads` kv heads at a time), formed twice, or the one for the short and the other for the long sequences of a batch.
struct Plan {
    uint32_t window, long_rows;
    struct Stored {
        uint32_t heads;          // 0: none
        uint32_t rows;           // M rows of a kv head that the scratch is laid out for
        uint32_t splits, split_len, pitch;
    } stored;
    struct Formed {
        uint32_t sequences;      // that may be formed twice (0: none)
        uint32_t rows, tiles, tiles_per_seq, splits, split_len;
    } formed;
    size_t bytes;                // (the parts of a call take turns in the same scratch)
};

Plan plan_of(uint32_t total_tokens, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t block_size, uint32_t batch,
             uint32_t max_num_block, uint32_t window)
{
    Plan plan{};
    plan.window = window = window >= total_tokens ? 0u : window;   // (as many rows as there are: all of them)
    const uint32_t G = n_heads / n_kv_heads, max_ctx = max_num_block * block_size;
    // counted rows: at most `window` per sequence, at most every row
    const uint64_t bounded = window == 0 ? total_tokens : static_cast<uint64_t>(window) * batch;
    const uint64_t counted = std::min<uint64_t>(bounded, total_tokens);
    if (counted * G <= static_cast<uint64_t>(kStoredRows) * batch && bounded * n_heads < (1ull << 31)) {
        const uint32_t rows = static_cast<uint32_t>(bounded) * G;
        const uint32_t pitch = ceil_div(max_ctx, 64u) * 64u;
        // what a kv head takes: a normaliser and a score a position for every row, two statistics for every 64 positions at the most
        const size_t of_head = rows * (static_cast<size_t>(pitch) + pitch / 32 + 1) * sizeof(float);
        uint32_t heads = static_cast<uint32_t>(std::min<size_t>(n_kv_heads, kStoredBytes / of_head));
        heads = heads < n_kv_heads && heads > kStoredWaves ? heads / kStoredWaves * kStoredWaves : heads;
        if (heads != 0) {
            plan.stored = {heads, rows, 0, 0, pitch};
            // chunks of 64 to 512 positions: the longest that leave 4096 waves (16 per compute unit; 12 fit)
            const uint64_t waves64 = static_cast<uint64_t>(batch) * ceil_div(max_ctx, 64u) * heads;
            plan.stored.split_len = static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>(8, waves64 / 4096))) * 64u;
            plan.stored.splits = ceil_div(max_ctx, plan.stored.split_len);
            const size_t all = static_cast<size_t>(rows) * heads;
            plan.bytes = ((all + 3) / 4 * 4 + all * pitch + 2 * all * plan.stored.splits) * sizeof(float);
            // how long a sequence may be while each of the others has a row. (Beside empty ones a longer one is possible: its scores
            // are stored like the others'. A call of one row a sequence must not pay for launches that find nothing to do.)
            const uint64_t others = batch - 1u, longest = total_tokens > others ? total_tokens - others : 1u;
            if ((window == 0 ? longest : std::min<uint64_t>(longest, window)) * G <= kLongRows) {
                return plan;
            }
            plan.long_rows = kLongRows;
        }
    }
    Plan::Formed &f = plan.formed;
    f.sequences = plan.long_rows == 0 ? batch : static_cast<uint32_t>(counted * G / (plan.long_rows + 1));   // (fewer than the batch: see the average)
    f.rows = total_tokens * G;
    const uint32_t tile = head_dim == 256 ? kRowTile / 2 : kRowTile;
    const uint64_t of_window = window == 0 ? 0 : static_cast<uint64_t>(std::min(window, total_tokens)) * G;
    f.tiles_per_seq = static_cast<uint32_t>((of_window + tile - 1) / tile);
    const uint32_t by_prefix = ceil_div(total_tokens * G, tile) + f.sequences;
    if (plan.long_rows == 0 && f.tiles_per_seq != 0 && static_cast<uint64_t>(f.tiles_per_seq) * batch <= by_prefix) {
        f.tiles = f.tiles_per_seq * batch;
    } else {
        f.tiles_per_seq = 0;
        f.tiles = by_prefix;
    }
    // splits of the row statistics: enough workgroups (of four waves) for four per compute unit
    const uint32_t want = ceil_div(2048u, std::max(1u, f.tiles * n_kv_heads));
    f.splits = std::max(1u, std::min(want, max_ctx / kMinSplit));
    f.split_len = ceil_div(ceil_div(max_ctx, f.splits), 32u) * 32u;
    const size_t rows = static_cast<size_t>(total_tokens) * n_heads;
    plan.bytes = std::max(plan.bytes, (rows + (f.splits > 1 ? 2 * f.splits * rows : 0)) * sizeof(float));
    return plan;
}

}  // namespace

}  // namespace xlite

using namespace xlite;

extern "C" size_t xlite_hip_attention_weights_workspace_bytes(uint32_t total_tokens, uint32_t n_heads, uint32_t n_kv_heads,
                                                              uint32_t head_dim, uint32_t block_size, uint32_t batch,
                                                              uint32_t max_num_block, uint32_t window)
{
    if (total_tokens == 0 || batch == 0 || n_kv_heads == 0 || n_heads == 0 || n_heads % n_kv_heads != 0) {
        return 0;
    }
    return plan_of(total_tokens, n_heads, n_kv_heads, head_dim, block_size, batch, max_num_block, window).bytes;
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
    XL_REQUIRE(aligned16(qkv) && aligned16(k_cache) && aligned16(workspace), "qkv, k_cache and workspace must be aligned to 16 bytes");
    const Plan plan = plan_of(total_tokens, n_heads, n_kv_heads, head_dim, block_size, batch, max_num_block, window);
    if (workspace == nullptr || workspace_bytes < plan.bytes) {
        return fail(XLITE_HIP_ENOSPC, __func__, "workspace too small: need " + std::to_string(plan.bytes) + " bytes, have " +
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
    p.window = plan.window;
    p.long_rows = plan.long_rows;
    p.block_magic = block_magic(block_size, max_ctx);
    p.norm = static_cast<float *>(workspace);
    // (16 splits of 2048 rows: 4.7 us either way; 251 of 16 rows: 64 us with a lane a row)
    auto join = [&](uint32_t rows, uint32_t splits) -> int {
        if (splits < 16) {
            join_stats_kernel<1><<<ceil_div(rows, 256u), 256, 0, s>>>(p.stats, p.norm, rows, splits);
        } else {
            join_stats_kernel<16><<<ceil_div(rows, 16u), 256, 0, s>>>(p.stats, p.norm, rows, splits);
        }
        XL_LAUNCH_CHECK();
        return XLITE_HIP_OK;
    };
    auto stored = [&](auto t, auto d, auto kvf) -> int {
        using T = decltype(t);
        constexpr int D = decltype(d)::value, KVF = decltype(kvf)::value;
        p.m_total = plan.stored.rows;
        p.splits = plan.stored.splits;
        p.split_len = plan.stored.split_len;
        p.pitch = plan.stored.pitch;
        const size_t lds = kStoredWaves * (StoredTile<D, KVF != XLITE_HIP_KV_SAME>::RING + stored_table(p.split_len, block_size) * sizeof(uint32_t));
        if (const int rc = ensure_dynamic_lds(reinterpret_cast<const void *>(store_scores_kernel<T, D, KVF>), lds)) {
            return rc;
        }
        for (p.head0 = 0; p.head0 < n_kv_heads; p.head0 += plan.stored.heads) {
            p.heads = std::min(plan.stored.heads, n_kv_heads - p.head0);
            const uint32_t rows = p.m_total * p.heads, heads = std::min(p.heads, kStoredWaves);
            p.scores = p.norm + (static_cast<size_t>(rows) + 3) / 4 * 4;   // (16-byte stores)
            p.stats = p.scores + static_cast<size_t>(rows) * p.pitch;
            store_scores_kernel<T, D, KVF><<<dim3(ceil_div(p.splits, kStoredWaves / heads) * ceil_div(p.heads, heads), batch),
                                             64 * kStoredWaves, lds, s>>>(p);
            XL_LAUNCH_CHECK();
            if (const int rc = join(rows, p.splits)) {
                return rc;
            }
            const uint32_t tiles = ceil_div(max_ctx, static_cast<uint32_t>(kThreads));
            const uint32_t z = std::max(1u, std::min(p.heads, 512u / std::max(1u, tiles * batch)));   // few positions: the heads side by side
            sum_scores_kernel<<<dim3(tiles, batch, z), kThreads, 0, s>>>(p);
            XL_LAUNCH_CHECK();
        }
        return XLITE_HIP_OK;
    };
    auto formed = [&](auto t, auto d, auto kvf) -> int {
        using T = decltype(t);
        constexpr int D = decltype(d)::value, KVF = decltype(kvf)::value;
        const Plan::Formed &f = plan.formed;
        const uint32_t rows = f.rows * n_kv_heads;
        p.m_total = f.rows;
        p.tiles_per_seq = f.tiles_per_seq;
        p.splits = f.splits;
        p.split_len = f.split_len;
        p.stats = p.norm + rows;
        // K through LDS: 16-bit caches whose copies (two positions of 256 elements, four of 128, eight of 64) lie in one block, and a
        // split's block-table entries behind the stages
        bool staged = false;
        if constexpr (KVF == XLITE_HIP_KV_SAME) {
            const size_t lds = 3 * kStagedPositions<D> * D * 2 + (static_cast<size_t>(p.split_len / block_size) + 2) * sizeof(uint32_t);
            staged = block_size % (512 / D) == 0 && p.block_magic != 0 && lds <= 64 * 1024;
            if (staged) {
                if (const int rc = ensure_dynamic_lds(reinterpret_cast<const void *>(row_stats_staged_kernel<T, D>), lds)) {
                    return rc;
                }
                row_stats_staged_kernel<T, D><<<dim3(f.tiles, p.splits, n_kv_heads), kThreads, lds, s>>>(p);
            }
        }
        if (!staged) {
            row_stats_kernel<T, D, KVF><<<dim3(f.tiles, p.splits, n_kv_heads), kThreads, 0, s>>>(p);
        }
        XL_LAUNCH_CHECK();
        if (p.splits > 1) {
            if (const int rc = join(rows, p.splits)) {
                return rc;
            }
        }
        const size_t lds = 3 * kTurns<D> * (32 * D * 2 + 4 * 256);
        if (const int rc = ensure_dynamic_lds(reinterpret_cast<const void *>(column_sums_kernel<T, D, KVF>), lds)) {
            return rc;
        }
        column_sums_kernel<T, D, KVF><<<dim3(ceil_div(max_ctx, 128u * kColumnTiles<D>), f.sequences, n_kv_heads), kTurns<D> * kThreads, lds, s>>>(p);
        XL_LAUNCH_CHECK();
        return XLITE_HIP_OK;
    };
    auto launch = [&](auto t, auto d, auto kvf) -> int {
        if (plan.stored.heads != 0) {
            if (const int rc = stored(t, d, kvf)) {
                return rc;
            }
        }
        return plan.formed.sequences != 0 ? formed(t, d, kvf) : XLITE_HIP_OK;
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
