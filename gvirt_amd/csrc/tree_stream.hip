// Attention over drafted trees: the cache streamed once, past all rows of a tree.
//
// A tree has few rows (nodes x query heads of a kv head: an M row each), so its attention is bound by reading K and V. The
// prefill kernel gives a workgroup one kv head: its copies are 256-byte rows up to two kilobytes apart, which memory serves
// at two thirds of the rate of longer runs, and four of its eight waves have no rows. Here a workgroup takes two kv heads
// times 128 M rows or one times 256, a wave 32 M rows of one head (the most that queries, results and operands
// leave registers for at two waves per SIMD), and copies of 1 KiB fetch the heads of a position together:
//     S^T[pos][m]  = K[pos][:] . Q[m][:]           v_mfma_f32_32x32x16 (A = K rows, ds_read_b128; B = Q)
//     O^T[d][m]   += V^T[d][pos] . P^T[pos][m]     v_mfma_f32_32x32x16 (A = V^T, ds_read_b64_tr_b16; B = P)
// Four stages of 32 KiB: one is consumed while three are on their way (with two of 64 KiB half of what memory delivers in a
// round trip was not asked for: a tenth slower for 64 trees of 32 over 8192 positions).
// Rows of less than 256 bytes: copied as they stand four steps ahead (caches of bytes: 18 KiB a step with their scales) and laid
// out in one of two stages, bytes widened to fp16; the scales join the scores. With the scales multiplied into fp16 rows an fp16 result was off by 5.5-8 e-4 of its size
// instead of 2.1 e-4 (its own rounding).
//
// Bound by memory where trees are small next to their contexts. Measured: 64 trees of 32 nodes over 8192 positions, 8 kv heads of
// 4, 2.19 GB: 402 us in the first calls after a pause, 440 once the clocks have settled under load (up to 640 on the way there), 5.4
// and 5.0 TB/s; 16 ragged trees of up to 27 over up to 4096, 170 MB: 49 us and 8 of merging. 8 trees of up to 16 over up to 16384
// int8 positions, 97 MB: 58 us and 8 of merging (the prefill kernel 80): 2 us a step of 16 KiB, the chain of widening, barrier,
// operands, scores, softmax and products. These trees fill two of the four row tiles of a head: the waves of the others only
// copy, so that one wave a SIMD computes. Half the vector instructions for widening, or the products of one half of the waves beside
// the widening of the other: the same time. head_dim 64, 16 bits: a tree of 8 over 700 positions 10 and 4 us (the prefill kernel
// 15), 64 ragged trees of 4 over 2000 25 us (31). head_dim 256: 32 ragged trees of 8 over 4000 positions of 4 heads, 330 MB: 64 us after a
// pause, 74 settled, and 5 of merging (the generic kernel 237).
//
// Work split: a sequence owns ceil(len G / rows) M tiles of ceil((cached + len) / step) steps each; the steps of all M tiles laid
// end to end are cut into equal chunks, one per workgroup, whatever the sequences' lengths (they live in device memory: every
// workgroup forms the prefix sums itself). A chunk that crosses an M tile's end runs as several segments. Chunk c owns the
// partial slots 2 c (its first segment) and 2 c + 1 (its last, when that is another one); an M tile cut into n segments from
// chunk c0 on finds them at 2 c0 (+ 1 unless it is that chunk's first), 2 (c0 + 1), ..., which its meta entry tells the merge.
#include <algorithm>
#include <type_traits>

#include "attention_common.h"
#include "block_magic.h"
#include "kv8.h"
#include "stage.h"

namespace xlite {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleSlack = 2.0f / kLog2e;   // the reference maximum moves when a score exceeds it by a factor of 4
constexpr int kRow = 128;                        // elements of a row in LDS
constexpr int kWaves = 8;
constexpr int kThreads = kWaves * 64;
constexpr uint32_t kHalf = 16 * 1024;            // K or V of a stage: 32 positions of two kv heads, 64 of one
constexpr uint32_t kStages = 4;
template <int NH>
constexpr uint32_t kRows = 32 * kWaves / NH;     // M rows of a workgroup, per kv head
constexpr uint32_t kStage = 2 * kHalf;
constexpr uint32_t kWaveRaw = 2 * 1024 + 256;    // short rows: what a wave copies in a step, 8 rows of K and of V and their scales
constexpr uint32_t kRawStage = kWaves * kWaveRaw;
constexpr uint32_t kScales = 3 * 64 * 4;         // of a widened stage: three numbers per (kv head, position)
template <bool RAW>
constexpr uint32_t kStageBytes = RAW ? 2 * (kStage + kScales) + kStages * kRawStage : kStages * kStage;
// Of a V row, in the arithmetic of its logarithm and reciprocal; the largest is its inverse. A row of the least scale beside one of the
// largest has its probability times 2^-100 in the exponential, which fp32 holds down to 2^-126, and gets the normaliser's share back.
constexpr float kLeastScale = 0x1p-50f;
constexpr uint32_t kTblCap = 2048;               // block-table entries staged per segment
constexpr uint32_t kSeqCap = 1024;               // sequences whose prefix sums fit
constexpr uint32_t kMaskCap = kThreads;          // mask words of an M tile kept in LDS: 128 rows of 4 heads and 512 nodes
constexpr uint32_t kMinChunk = 4;                // steps
constexpr uint32_t kComputeUnits = 256;

typedef __attribute__((__vector_size__(4 * sizeof(short)))) short s16x4_t;

template <typename T>
__device__ __forceinline__ f32x16_t mfma32(const uint4 &a, const uint4 &b, f32x16_t c)
{
    if constexpr (T::kCode == XLITE_HIP_BF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    }
}

struct StreamParams {
    const uint16_t *q;
    const unsigned char *k_cache;
    const unsigned char *v_cache;
    const float *k_scale;  // caches of bytes: [slot][kv head]
    const float *v_scale;
    uint16_t *out;
    const uint32_t *tree_mask;
    const int32_t *query_start_loc;
    const int32_t *lens;
    const int32_t *cached_lens;
    const int32_t *block_tables;
    int4 *meta;            // [M tile id]: segments to merge (0: the results are final), first chunk, first-segment flag
    float *acc;            // [head group][slot][kv head of the group][M rows of a tile][D], not normalised
    float *ml;             // the same without D: reference maximum (log2 domain), normaliser
    uint32_t q_tok_stride, n_heads, n_kv_heads, group;
    uint32_t batch, block_size, block_magic, max_num_block, mask_words;
    uint32_t slots;        // 2 x chunks a launch may have
};

// M tile ids of a sequence: floor(start * G / rows) + i on, at least as many as it has M tiles
template <int NH>
__device__ __forceinline__ uint32_t first_id(const StreamParams &p, uint32_t start, uint32_t seq)
{
    return static_cast<uint32_t>(static_cast<uint64_t>(start) * p.group / kRows<NH>) + seq;
}
__device__ __forceinline__ uint32_t uni(uint32_t x)
{
    return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x)));
}

// NH: kv heads of a workgroup. T: the type of the products; TIO: of the query rows and the output (the same, or bf16 with fp16
// products over caches of bytes, KVF). Rows shorter than
// 256 bytes (caches of bytes, D = 64) are copied as they are and laid out by the wave that copied them; of D = 64, half of a
// row in LDS is not used.
// WIDE: head_dim 256, as two heads of 128 in memory whose scores are added: a wave forms the scores of both halves and the
// results of one.
template <typename T, int NH, int KVF, typename TIO, int D, bool WIDE>
__global__ void __launch_bounds__(kThreads, 1)
tree_stream_kernel(const StreamParams p)
{
    static_assert(!WIDE || (NH == 2 && D == 128 && KVF == XLITE_HIP_KV_SAME), "two halves of 128 elements, 16-bit caches");
    constexpr bool KV8 = KVF != XLITE_HIP_KV_SAME, RAW = KV8 || D == 64;
    static_assert(D == 128 || D == 64, "head_dim 64 or 128");
    constexpr int KS = D / 16, DT = D / 32, HALVES = WIDE ? 2 : 1;
    constexpr uint32_t ROWS = kRows<NH>;
    constexpr uint32_t POSB = NH * 256;          // LDS bytes of a position
    constexpr uint32_t SP = kHalf / POSB;        // positions of a step
    constexpr uint32_t PPI = 1024 / POSB;        // positions of a copy
    constexpr int CPW = 2;                       // copies per wave, step and tensor
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    uint32_t *tbl = reinterpret_cast<uint32_t *>(smem + kStageBytes<RAW>);
    uint32_t *mask_lds = tbl + kTblCap;
    uint32_t *pref = mask_lds + kMaskCap;        // batch + 1 words
    const uint32_t smem_addr = stage::lds_address(smem);
    const uint32_t lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
    const uint32_t G = p.group;
    const uint32_t hsel = wave % NH, row_tile = wave / NH;
    const uint32_t kvh = blockIdx.y * NH + hsel;

    // ---- steps of every sequence, summed. Up to 64 sequences: lane i of every wave holds what the batch says about sequence
    // i (one round of loads, nothing through LDS); more: thread t owns consecutive sequences and the sums go to LDS.
    auto weight = [&](int32_t n, int32_t c) {
        return n <= 0 ? 0u : ceil_div(static_cast<uint32_t>(c + n), SP) * ceil_div(static_cast<uint32_t>(n) * G, ROWS);
    };
    const bool in_lanes = p.batch <= 64;
    int32_t ln_len = 0, ln_cached = 0, ln_start = 0;
    uint32_t ln_pref = 0, total;
    if (in_lanes) {
        const uint32_t i = min(lane, p.batch - 1);
        ln_len = p.lens[i];
        ln_cached = p.cached_lens[i];
        ln_start = p.query_start_loc[i];
        uint32_t incl = lane < p.batch ? weight(ln_len, ln_cached) : 0u;
        const uint32_t mine = incl;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t up = __shfl_up(incl, d);
            incl += lane >= static_cast<uint32_t>(d) ? up : 0u;
        }
        ln_pref = incl - mine;   // (lanes past the batch: the sum of everything)
        total = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(incl), 63));
    } else {
        const uint32_t per = ceil_div(p.batch, static_cast<uint32_t>(kThreads));
        const uint32_t i0 = min(p.batch, threadIdx.x * per), i1 = min(p.batch, i0 + per);
        uint32_t mine = 0;
        for (uint32_t i = i0; i < i1; i++) {
            mine += weight(p.lens[i], p.cached_lens[i]);
        }
        uint32_t incl = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t up = __shfl_up(incl, d);
            incl += lane >= static_cast<uint32_t>(d) ? up : 0u;
        }
        if (lane == 63) {
            tbl[wave] = incl;   // (the table's words are not in use yet)
        }
        __syncthreads();
        uint32_t run = incl - mine;
        for (uint32_t w = 0; w < wave; w++) {
            run += tbl[w];
        }
        for (uint32_t i = i0; i < i1; i++) {
            pref[i] = run;
            run += weight(p.lens[i], p.cached_lens[i]);
        }
        if (threadIdx.x == kThreads - 1) {
            pref[p.batch] = run;
        }
        __syncthreads();
        total = uni(pref[p.batch]);
    }
    auto steps_before = [&](uint32_t i) {   // sequence i; i == batch: all of them
        return in_lanes ? (i < 64 ? static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(ln_pref), static_cast<int>(i))) : total) : uni(pref[i]);
    };
    uint32_t chunk = max(ceil_div(total, gridDim.x), kMinChunk);
    chunk = min(chunk, (kTblCap - 2) * p.block_size / SP);
    const uint32_t n_chunks = ceil_div(total, chunk);

    // ---- read roles (the pattern of position p + 32 is that of p)
    const uint32_t k_off = col * POSB + (WIDE ? 0u : hsel * 256);
    const uint32_t kx = (half ^ stage::pattern<kRow>(col)) << 4;
    uint32_t v_off;
    {
        const uint32_t g = lane >> 4, jp = (lane & 15) >> 2, q = lane & 3;
        const uint32_t y = 2 * (g & 1) + (q >> 1), pos = 4 * (g >> 1) + jp;
        v_off = kHalf + pos * POSB + hsel * 256 + ((y ^ stage::pattern<kRow>(pos)) << 4) + ((q & 1) << 3);
    }
    // ---- copy role: wave w fills copies 2 w and 2 w + 1 of the K and of the V half. Lane l of a copy: row l / 16 of its four
    // (position, kv head) rows, chunk slot l % 16, which receives chunk slot ^ pattern(position)
    const uint32_t row_bytes = p.n_kv_heads * 256;
    for (uint32_t c = blockIdx.x; c < n_chunks; c += gridDim.x) {
        const uint32_t c_begin = c * chunk, c_end = min(total, c_begin + chunk);
        uint32_t at = c_begin;
        uint32_t seq = 0;   // the last sequence whose first step is at or before `at`
        if (in_lanes) {
            seq = static_cast<uint32_t>(__builtin_popcountll(__ballot(lane < p.batch && ln_pref <= at))) - 1;
        } else {
            uint32_t hi = p.batch;
            while (hi - seq > 1) {
                const uint32_t mid = (seq + hi) >> 1;
                if (uni(pref[mid]) <= at) {
                    seq = mid;
                } else {
                    hi = mid;
                }
            }
        }
        while (at < c_end) {
            seq = uni(seq);
            const uint32_t first = steps_before(seq), next = steps_before(seq + 1);
            if (next == first) {   // no rows
                seq++;
                continue;
            }
            // ---- the segment: steps a .. b - 1 of M tile mt
            const int32_t at_lane = static_cast<int>(min(seq, 63u));
            const uint32_t nodes = uni(static_cast<uint32_t>(in_lanes ? __builtin_amdgcn_readlane(ln_len, at_lane) : p.lens[seq]));
            const uint32_t cached = uni(static_cast<uint32_t>(in_lanes ? __builtin_amdgcn_readlane(ln_cached, at_lane) : p.cached_lens[seq]));
            const uint32_t start = uni(static_cast<uint32_t>(in_lanes ? __builtin_amdgcn_readlane(ln_start, at_lane) : p.query_start_loc[seq]));
            const uint32_t range = cached + nodes, steps = ceil_div(range, SP);
            const uint32_t mt = (at - first) / steps, a = (at - first) - mt * steps, b = min(steps, a + (c_end - at));
            const uint32_t tile_first = first + mt * steps;      // of the M tile, in all steps
            const bool whole = a == 0 && b == steps;
            const bool first_seg = at == c_begin;
            const uint32_t id = first_id<NH>(p, start, seq) + mt;
            const uint32_t m_rows = nodes * G, m_first = mt * ROWS + row_tile * 32;   // (the wave's first)
            const bool has_rows = m_first < m_rows;
            const uint32_t m = min(m_first + col, m_rows - 1);       // (rows past the end repeat the last one, unstored)
            const uint64_t tok = start + m / G;
            const uint32_t head = (WIDE ? blockIdx.y : kvh) * G + m % G;
            const uint32_t t0 = a * SP, t1 = min(range, b * SP);
            const int32_t *table = p.block_tables + static_cast<uint64_t>(seq) * p.max_num_block;
            const uint32_t blk0 = t0 / p.block_size, blk1 = (t1 - 1) / p.block_size;

            // ---- set-up: block-table entries, then the query rows, then the first steps' copies
            __syncthreads();   // (the table and the stages of the last segment have been read)
            const uint32_t n_blk = blk1 - blk0 + 1;
            // the mask's rows of the M tile, for a segment that reaches into the tree
            const uint32_t tok_first = mt * ROWS / G;                   // (inside the sequence)
            const uint32_t tok_count = (min(mt * ROWS + ROWS, m_rows) - 1) / G - tok_first + 1;
            const uint32_t n_words = tok_count * p.mask_words;
            const bool words_in_lds = n_words <= kMaskCap;
            const uint32_t *words_src = p.tree_mask + static_cast<uint64_t>(start + tok_first) * p.mask_words;
            const uint32_t word = words_src[words_in_lds ? min(threadIdx.x, n_words - 1) : 0u];
            const uint32_t entry = static_cast<uint32_t>(table[blk0 + min(threadIdx.x, n_blk - 1)]);
            uint4 qreg[HALVES * KS];
            const uint16_t *src = p.q + tok * p.q_tok_stride + static_cast<uint64_t>(head) * (HALVES * D);
#pragma unroll
            for (int ks = 0; ks < HALVES * KS; ks++) {
                qreg[ks] = *reinterpret_cast<const uint4 *>(src + ks * 16 + half * 8);
            }
            // (this wait leaves the query rows on their way)
            if (words_in_lds && threadIdx.x < n_words) {
                mask_lds[threadIdx.x] = word;
            }
            if (threadIdx.x < n_blk) {
                tbl[threadIdx.x] = entry;
            }
            for (uint32_t i = threadIdx.x + kThreads; i < n_blk; i += kThreads) {
                tbl[i] = static_cast<uint32_t>(table[blk0 + i]);
            }
            if (a == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
                const uint32_t n = whole ? 0u : (tile_first + steps - 1) / chunk - c + 1;
                p.meta[id] = make_int4(static_cast<int>(n), static_cast<int>(c), first_seg ? 1 : 0, 0);
            }
            f32x16_t O[DT];
            float m_run = -INFINITY, l_run = 0.f;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    O[dt][k] = 0.f;
                }
            }
            __syncthreads();
            // copies of step `s` (from t0) into stage s % 4. Positions at or beyond t1 re-read the last one (their scores are
            // masked). The positions of a copy share a block, and if blocks are multiples of all of a wave's, those do.
            const bool one_block = p.block_size % (CPW * PPI) == 0;
            auto issue = [&](uint32_t s) __attribute__((always_inline)) {
                const uint32_t base_pos = t0 + s * SP + CPW * wave * PPI;
                const uint32_t st = smem_addr + (s % kStages) * kStage + wave * (CPW * 1024);
                const char *kc = reinterpret_cast<const char *>(p.k_cache) + blockIdx.y * (NH * 256);
                const char *vc = reinterpret_cast<const char *>(p.v_cache) + blockIdx.y * (NH * 256);
                // (worked out anew in every step, from a lane number that the compiler cannot carry along: a register spilled
                // in this loop is reloaded by a memory load, whose wait is for every copy on its way)
                uint32_t l = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
                asm volatile("" : "+v"(l));
                const uint32_t c_rel = (l >> 4) / NH, c_head = (l >> 4) % NH;
                auto c_off = [&](int i) __attribute__((always_inline)) {
                    const uint32_t pos = (CPW * wave + i) * PPI + c_rel;
                    return c_head * 256 + (((l & 15u) ^ stage::pattern<kRow>(pos)) << 4);
                };
                if (one_block && base_pos + CPW * PPI <= t1) {
                    const uint32_t blk = __umulhi(base_pos, p.block_magic);
                    const uint32_t phys = uni(tbl[blk - blk0]);
                    const uint64_t row0 = static_cast<uint64_t>(phys) * p.block_size + (base_pos - blk * p.block_size);
                    const char *kb = kc + row0 * row_bytes, *vb = vc + row0 * row_bytes;
#pragma unroll
                    for (int i = 0; i < CPW; i++) {
                        stage::copy_1k_once(st + i * 1024, c_off(i) + c_rel * row_bytes, kb + static_cast<uint32_t>(i * PPI) * row_bytes);
                    }
#pragma unroll
                    for (int i = 0; i < CPW; i++) {
                        stage::copy_1k_once(st + kHalf + i * 1024, c_off(i) + c_rel * row_bytes, vb + static_cast<uint32_t>(i * PPI) * row_bytes);
                    }
                    return;
                }
#pragma unroll
                for (int i = 0; i < CPW; i++) {
                    const uint32_t t_raw = base_pos + i * PPI;
                    const uint32_t t = min(t_raw, t1 - 1) & ~(PPI - 1);
                    const uint32_t rel = min(t_raw + c_rel, t1 - 1) - t;
                    const uint32_t blk = __umulhi(t, p.block_magic);
                    const uint32_t phys = uni(tbl[blk - blk0]);
                    const uint64_t row0 = static_cast<uint64_t>(phys) * p.block_size + (t - blk * p.block_size);
                    const char *kb = kc + row0 * row_bytes, *vb = vc + row0 * row_bytes;
                    stage::copy_1k_once(st + i * 1024, c_off(i) + rel * row_bytes, kb);
                    stage::copy_1k_once(st + kHalf + i * 1024, c_off(i) + rel * row_bytes, vb);
                }
            };

            // Short rows: a wave copies 8 (position, kv head) rows of K and of V (and the scales of bytes) per step, four steps
            // ahead, and lays out what it copied itself as the rows of one of two stages, bytes widened to fp16: no barrier in
            // between. The bytes' values are exact in fp16 and the scales stay in fp32: K's multiplies the scores, V's goes into the
            // exponents (p vs = 2^(x + log2 vs), rounded once, in range whatever the scales) and out of the normaliser.
            constexpr uint32_t RP = 8 / NH;                 // positions of a wave
            constexpr uint32_t ROWM = KV8 ? D : 2 * D;      // bytes of a row in memory: 64 or 128 here
            constexpr uint32_t COPIES = ROWM == 64 ? 1 : 2; // of 1 KiB: both tensors in one, or one each
            constexpr uint32_t OPS = COPIES + (KV8 ? 1 : 0);
            auto row8 = [&](uint32_t s, uint32_t r) __attribute__((always_inline)) {
                const uint32_t pos = min(t0 + s * SP + wave * RP + r / NH, t1 - 1), blk = __umulhi(pos, p.block_magic);
                return (static_cast<uint64_t>(tbl[blk - blk0]) * p.block_size + (pos - blk * p.block_size)) * p.n_kv_heads + blockIdx.y * NH + r % NH;
            };
            constexpr uint32_t RING = 2 * (kStage + kScales);
            auto issue8 = [&](uint32_t s) __attribute__((always_inline)) {
                const uint32_t st = smem_addr + RING + (s % kStages) * kRawStage + wave * kWaveRaw;
                if constexpr (COPIES == 2) {
                    const uint64_t off = row8(s, lane >> 3) * ROWM + (lane & 7u) * 16;
                    stage::copy_lanes_16_once(st, p.k_cache + off);
                    stage::copy_lanes_16_once(st + 1024, p.v_cache + off);
                } else {
                    stage::copy_lanes_16_once(st, (half != 0 ? p.v_cache : p.k_cache) + row8(s, (lane >> 2) & 7u) * ROWM + (lane & 3u) * 16);
                }
                if constexpr (KV8) {   // K: words 0 .. 7, V: 8 .. 15
                    stage::copy_lanes_4(st + 2048, ((lane & 8u) != 0 ? p.v_scale : p.k_scale) + row8(s, lane & 7u));
                }
            };
            auto lay_out = [&](uint32_t s) __attribute__((always_inline)) {
                const unsigned char *raw = smem + RING + (s % kStages) * kRawStage + wave * kWaveRaw;
                unsigned char *st = smem + (s % 2) * kStage;
                const uint32_t r = COPIES == 2 ? lane >> 3 : (lane >> 2) & 7u, c = COPIES == 2 ? lane & 7u : lane & 3u;   // row, 16 bytes of it
                const uint32_t pos = wave * RP + r / NH, x = stage::pattern<kRow>(pos);
                unsigned char *dst = st + pos * POSB + (r % NH) * 256 + (COPIES == 2 ? 0u : half * kHalf);
#pragma unroll
                for (uint32_t v = 0; v < COPIES; v++) {
                    const uint4 bytes = *reinterpret_cast<const uint4 *>(raw + v * 1024 + lane * 16);
                    if constexpr (KV8) {
                        *reinterpret_cast<uint4 *>(dst + v * kHalf + (((2 * c) ^ x) << 4)) = widen8<KVF>(make_uint2(bytes.x, bytes.y));
                        *reinterpret_cast<uint4 *>(dst + v * kHalf + (((2 * c + 1) ^ x) << 4)) = widen8<KVF>(make_uint2(bytes.z, bytes.w));
                    } else {
                        *reinterpret_cast<uint4 *>(dst + v * kHalf + ((c ^ x) << 4)) = bytes;
                    }
                }
                if (KV8 && lane < 16) {
                    const float scale = *reinterpret_cast<const float *>(raw + 2048 + lane * 4);
                    const uint32_t rs = lane & 7u;
                    float *to = reinterpret_cast<float *>(smem + 2 * kStage + (s % 2) * kScales) + (rs % NH) * SP + wave * RP + rs / NH;
                    if (lane < 8) {
                        to[0] = scale * kLog2e;
                    } else {
                        const float vs = fminf(fmaxf(scale, kLeastScale), 1.0f / kLeastScale);
                        to[64] = scale != scale ? scale : __log2f(vs);   // (a NaN: of the scores, so that only rows that see it get it)
                        to[128] = 1.0f / vs;
                    }
                }
            };

            // which of the positions j0 .. j0 + 31 the lane's row sees, moved so that bit 8 (k / 4) + k % 4 is that of register k
            auto seen_from = [&](uint32_t j0) __attribute__((always_inline)) {
                const uint32_t *words = words_in_lds ? mask_lds + (m / G - tok_first) * p.mask_words : p.tree_mask + tok * p.mask_words;
                return (tree_seen(words, p.mask_words, j0, cached, nodes) & ones(static_cast<int32_t>(t1 - j0))) >> (4 * half);
            };
            bool poisoned = false;
            // 32 positions of a step: those from 32 h on. Register k of S holds position j0 + 8 (k / 4) + 4 half + k % 4.
            auto compute = [&](uint32_t s, uint32_t h) __attribute__((always_inline)) {
                const uint32_t j0 = t0 + s * SP + 32 * h;
                const bool masked = j0 + 32 > cached;   // (positions below the cached length are seen by every row)
                const unsigned char *st = smem + (s % (RAW ? 2 : kStages)) * kStage + h * 32 * POSB;
                f32x16_t S;
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    S[k] = 0.f;
                }
#pragma unroll
                for (int w = 0; w < HALVES; w++) {
                    uint4 kop[KS];
#pragma unroll
                    for (int ks = 0; ks < KS; ks++) {
                        kop[ks] = *reinterpret_cast<const uint4 *>(st + k_off + w * 256 + (((2 * ks) << 4) ^ kx));
                    }
#pragma unroll
                    for (int ks = 0; ks < KS; ks++) {
                        S = mfma32<T>(kop[ks], qreg[w * KS + ks], S);
                    }
                    if (WIDE) {
                        __builtin_amdgcn_sched_barrier(0);   // (the operands of one half at a time: the registers hold no more)
                    }
                }
                // V^T operands: on their way during the softmax
                typedef s16x4_t __attribute__((address_space(3))) * lds_tr_ptr;
                unsigned char *vbase = const_cast<unsigned char *>(st);
                uint4 vop[2][DT];
#pragma unroll
                for (int kk = 0; kk < 2; kk++) {
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) {
                        const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (lds_tr_ptr)(vbase + kk * 16 * POSB + (v_off ^ (dt << 6)))));
                        // 8 positions further: the pattern of position p + 8 is that of p XOR 2
                        const uint2 hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (lds_tr_ptr)(vbase + (kk * 16 + 8) * POSB + (v_off ^ ((dt << 6) | (1 << 5))))));
                        vop[kk][dt] = make_uint4(lo.x, lo.y, hi.x, hi.y);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                [[maybe_unused]] const float *scales = reinterpret_cast<const float *>(smem + 2 * kStage + (s % 2) * kScales) + hsel * SP + 32 * h + 4 * half;
                if constexpr (KV8) {   // in units of log2, with V's scale
#pragma unroll
                    for (int kg = 0; kg < 4; kg++) {
                        const float4 ks = *reinterpret_cast<const float4 *>(scales + 8 * kg), lv = *reinterpret_cast<const float4 *>(scales + 64 + 8 * kg);
                        S[4 * kg] = __builtin_fmaf(S[4 * kg], ks.x, lv.x);
                        S[4 * kg + 1] = __builtin_fmaf(S[4 * kg + 1], ks.y, lv.y);
                        S[4 * kg + 2] = __builtin_fmaf(S[4 * kg + 2], ks.z, lv.z);
                        S[4 * kg + 3] = __builtin_fmaf(S[4 * kg + 3], ks.w, lv.w);
                    }
                }
                if (masked) {
                    uint32_t seen = seen_from(j0);
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        S[k] = (seen >> ((k / 4) * 8 + (k % 4))) & 1u ? S[k] : -INFINITY;
                    }
                    // A row that does not see a position has probability zero there, and zero times an infinity or a NaN in
                    // that position's V row would still poison it. Such values leave the operands; the rows that see them
                    // get them back behind the loop. (Values widened from bytes are finite.)
                    uint32_t odd = 0;
#pragma unroll
                    for (int kk = 0; kk < (KV8 ? 0 : 2); kk++) {
#pragma unroll
                        for (int dt = 0; dt < DT; dt++) {
                            odd |= not_finite2<T>(vop[kk][dt].x) | not_finite2<T>(vop[kk][dt].y) | not_finite2<T>(vop[kk][dt].z) |
                                   not_finite2<T>(vop[kk][dt].w);
                        }
                    }
                    if (!KV8 && __any(odd)) {
                        poisoned = true;
#pragma unroll
                        for (int kk = 0; kk < 2; kk++) {
#pragma unroll
                            for (int dt = 0; dt < DT; dt++) {
                                vop[kk][dt] = make_uint4(finite_only<T>(vop[kk][dt].x), finite_only<T>(vop[kk][dt].y),
                                                         finite_only<T>(vop[kk][dt].z), finite_only<T>(vop[kk][dt].w));
                            }
                        }
                    }
                }
                float mx = -INFINITY;
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    mx = fmaxf(mx, S[k]);
                }
                {
                    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
                    mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
                }
                // (the reference moves only when exceeded by more than a factor of 4, as in the prefill kernel)
                const float m_new = mx > m_run + (KV8 ? 2.0f : kRescaleSlack) ? mx : m_run;
                const float m_safe = m_new == -INFINITY ? 0.f : m_new;
                const float alpha = fast_exp2((m_run - m_safe) * (KV8 ? 1.0f : kLog2e));
                const float neg_m = -m_safe * kLog2e;
                m_run = m_new;
                uint32_t w[8];
                float psum = 0.f;
#pragma unroll
                for (int k = 0; k < 16; k += 2) {
                    float e0, e1;
                    if constexpr (KV8) {
                        e0 = fast_exp2(S[k] - m_safe);
                        e1 = fast_exp2(S[k + 1] - m_safe);
                        const float2 inv = *reinterpret_cast<const float2 *>(scales + 128 + (k / 4) * 8 + k % 4);
                        psum = __builtin_fmaf(e0, inv.x, psum);
                        psum = __builtin_fmaf(e1, inv.y, psum);
                    } else {
                        e0 = fast_exp2(__builtin_fmaf(S[k], kLog2e, neg_m));
                        e1 = fast_exp2(__builtin_fmaf(S[k + 1], kLog2e, neg_m));
                        psum += e0 + e1;
                    }
                    w[k / 2] = T::pack(e0, e1);   // rounded to the products' type: half a step of it, 2^-8 (2^-11) of each
                }
                const uint4 pb[2] = {make_uint4(w[0], w[1], w[2], w[3]), make_uint4(w[4], w[5], w[6], w[7])};
                l_run = l_run * alpha + psum;
                if (__any(alpha != 1.0f)) {
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) {
#pragma unroll
                        for (int k = 0; k < 16; k++) {
                            // (in place: an opaque multiply keeps the accumulators in the same registers on both paths)
                            asm volatile("v_mul_f32 %0, %1, %0" : "+v"(O[dt][k]) : "v"(alpha));
                        }
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int kk = 0; kk < 2; kk++) {
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) {
                        O[dt] = mfma32<T>(vop[kk][dt], pb[kk], O[dt]);
                    }
                }
            };

            const uint32_t n_steps = b - a, last = n_steps - 1;
            if constexpr (RAW) {
                for (uint32_t s = 0; s < min(n_steps, kStages); s++) {
                    issue8(s);
                }
            } else {
                issue(0);
                if (last >= 1) {
                    issue(1);
                }
                if (last >= 2) {
                    issue(2);
                }
            }
            // (the query rows were requested before the copies; their wait is for both)
#pragma unroll
            for (int ks = 0; ks < HALVES * KS; ks++) {
                asm volatile("" : "+v"(qreg[ks].x), "+v"(qreg[ks].y), "+v"(qreg[ks].z), "+v"(qreg[ks].w));
                qreg[ks] = convert8<TIO, T>(qreg[ks]);
            }
            for (uint32_t s = 0; s < n_steps; s++) {
                if constexpr (RAW) {
                    // this wave's share of step s has landed: OPS of each of the next three steps are out
                    if (s + 3 <= last) {
                        stage::wait<3 * OPS>();
                    } else if (s + 2 <= last) {
                        stage::wait<2 * OPS>();
                    } else if (s + 1 <= last) {
                        stage::wait<OPS>();
                    } else {
                        stage::wait<0>();
                    }
                    lay_out(s);          // (the stage of step s - 2: everybody was past it at the barrier of step s - 1)
                    __syncthreads();
                    if (s + 4 <= last) {
                        issue8(s + 4);
                    }
                    if (has_rows) {
#pragma unroll 1
                        for (uint32_t h = 0; h < SP / 32; h++) {
                            compute(s, h);
                        }
                    }
                    continue;
                }
                // this wave's share of step s has landed: only those of the next two are out
                if (s + 2 <= last) {
                    stage::wait<4 * CPW>();
                } else if (s + 1 <= last) {
                    stage::wait<2 * CPW>();
                } else {
                    stage::wait<0>();
                }
                __syncthreads();   // ... and everybody else's; the stage of step s - 1 is free
                if (s + 3 <= last) {
                    issue(s + 3);
                }
                if (has_rows) {    // (a wave without rows only copies)
#pragma unroll 1
                    for (uint32_t h = 0; h < SP / 32; h++) {
                        compute(s, h);
                    }
                }
            }
            if (!KV8 && poisoned) {   // (rare, and not fast: the V rows of the masked steps are read again, value by value)
                // from the first masked step on, whose positions below the cached length every row sees (segments begin at
                // multiples of 32 positions, as the halves of a step do)
                for (uint32_t j = max(t0, cached & ~31u); j < t1; j++) {
                    const uint32_t blk = j / p.block_size;
                    const uint64_t row = static_cast<uint64_t>(static_cast<uint32_t>(table[blk])) * p.block_size + (j - blk * p.block_size);
                    const uint16_t *v = reinterpret_cast<const uint16_t *>(p.v_cache) + (row * p.n_kv_heads + kvh) * D + 4 * half;
                    const bool see = tree_seen(p.tree_mask + tok * p.mask_words, p.mask_words, j, cached, nodes) & 1u;
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) {
#pragma unroll
                        for (int k = 0; k < 16; k++) {
                            const uint32_t bits = v[dt * 32 + (k / 4) * 8 + (k % 4)];
                            const float x = T::to_f32(static_cast<uint16_t>(bits));
                            O[dt][k] += see && not_finite2<T>(bits) ? x : 0.f;
                        }
                    }
                }
            }
            // ---- results. O^T lane layout: column = M row, register k of tile dt = element 32 dt + 8 (k / 4) + 4 half + k % 4
            const float l_tot = l_run + __shfl_xor(l_run, 32);
            if (m_first + col < m_rows) {
                if (whole) {
                    const float inv = l_tot > 0.f ? 1.0f / l_tot : 0.f;   // (NaN is not above 0 ...)
                    const float scale = l_tot != l_tot ? l_tot : inv;     // (... and stays NaN)
                    uint16_t *dst = p.out + (tok * p.n_heads + head) * (HALVES * D) + (WIDE ? hsel * D : 0u);
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) {
#pragma unroll
                        for (int kg = 0; kg < 4; kg++) {
                            uint2 o;
                            o.x = TIO::pack(O[dt][kg * 4] * scale, O[dt][kg * 4 + 1] * scale);
                            o.y = TIO::pack(O[dt][kg * 4 + 2] * scale, O[dt][kg * 4 + 3] * scale);
                            *reinterpret_cast<uint2 *>(dst + dt * 32 + kg * 8 + half * 4) = o;
                        }
                    }
                } else {
                    const uint64_t slot = static_cast<uint64_t>(blockIdx.y) * p.slots + 2 * c + (first_seg ? 0u : 1u);
                    // as the registers lie: 16 pieces of 1 KiB per 32 rows, piece 4 dt + kg lane by lane
                    const uint64_t tile = (slot * NH + hsel) * (ROWS / 32) + row_tile;
                    float4 *dst = reinterpret_cast<float4 *>(p.acc + tile * 32 * D) + lane;
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) {
#pragma unroll
                        for (int kg = 0; kg < 4; kg++) {
                            dst[(dt * 4 + kg) * 64] = make_float4(O[dt][kg * 4], O[dt][kg * 4 + 1], O[dt][kg * 4 + 2], O[dt][kg * 4 + 3]);
                        }
                    }
                    if (half == 0) {
                        *reinterpret_cast<float2 *>(p.ml + (tile * 32 + col) * 2) = make_float2(KV8 ? m_run : m_run * kLog2e, l_tot);
                    }
                }
            }
            at += b - a;
            if (at >= next) {
                seq++;
            }
        }
    }
}

// Joins the partials of an M tile: a workgroup per (M tile, kv head, 16 rows), D / 8 threads of 8 columns (a piece of the stored
// layout) per row, and TURNS such sets that take the segments in turn.
template <typename T, int NH, int D, int TURNS, bool WIDE>
__global__ void __launch_bounds__(2 * D * TURNS)
tree_merge_kernel(const StreamParams p)
{
    constexpr int U = TURNS > 1 ? 8 : 4;   // segments of a set at a time
    __shared__ float part[TURNS > 1 ? TURNS - 1 : 1][10][2 * D];
    const uint32_t id = blockIdx.x, kvh = blockIdx.y, G = p.group;
    const uint32_t turn = threadIdx.x / (2 * D), in_set = threadIdx.x % (2 * D);
    uint32_t seq = 0;   // the last sequence whose ids start at or before `id`
    int32_t n;
    uint32_t start;
    const int4 meta = p.meta[id];
    if (p.batch <= 64) {   // one round of loads
        const uint32_t lane = threadIdx.x & 63, i = min(lane, p.batch - 1);
        const int32_t ln_start = p.query_start_loc[i], ln_len = p.lens[i];
        const uint64_t started = __ballot(lane < p.batch && first_id<NH>(p, static_cast<uint32_t>(ln_start), lane) <= id);
        seq = static_cast<uint32_t>(max(__builtin_popcountll(started) - 1, 0));
        n = __shfl(ln_len, static_cast<int>(seq));
        start = static_cast<uint32_t>(__shfl(ln_start, static_cast<int>(seq)));
    } else {
        uint32_t hi = p.batch;
        while (hi - seq > 1) {
            const uint32_t mid = (seq + hi) >> 1;
            if (first_id<NH>(p, static_cast<uint32_t>(p.query_start_loc[mid]), mid) <= id) {
                seq = mid;
            } else {
                hi = mid;
            }
        }
        n = p.lens[seq];
        start = static_cast<uint32_t>(p.query_start_loc[seq]);
    }
    const uint32_t mt = id - first_id<NH>(p, start, seq), m_rows = static_cast<uint32_t>(max(n, 0)) * G;
    const uint32_t m_first = mt * kRows<NH> + blockIdx.z * 16;
    if (m_first >= m_rows) {   // (the whole workgroup)
        return;
    }
    const uint32_t segments = static_cast<uint32_t>(meta.x);
    const bool shared = TURNS > 1 && segments > U;   // by the sets
    if (segments == 0 || (turn != 0 && !shared)) {
        return;
    }
    const uint32_t in_tile = blockIdx.z * 16 + in_set % 16, m = mt * kRows<NH> + in_tile;   // (rows past the end: partials of no row, unstored)
    const uint32_t c0 = static_cast<uint32_t>(meta.y), first = static_cast<uint32_t>(meta.z), piece = in_set / 16;
    const uint64_t group0 = static_cast<uint64_t>(kvh / NH) * p.slots;
    auto row_of = [&](uint32_t s) {
        const uint64_t slot = group0 + (s == 0 ? 2 * c0 + (1 - first) : 2 * (c0 + s));
        return (slot * NH + kvh % NH) * kRows<NH> + in_tile;
    };
    float m_all = -INFINITY, l = 0.f, o[8] = {};
    auto join = [&](float m_part, float l_part, const float (&x)[8]) __attribute__((always_inline)) {
        const float m_new = fmaxf(m_all, m_part), safe = m_new == -INFINITY ? 0.f : m_new;
        const float wa = fast_exp2(m_all - safe), wb = fast_exp2(m_part - safe);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            o[e] = o[e] * wa + (wb != 0.f ? x[e] * wb : 0.f);   // (a part of weight zero that saw nothing holds zeros)
        }
        l = l * wa + l_part * wb;
        m_all = m_new;
    };
    for (uint32_t i0 = U * turn; i0 < segments; i0 += U * TURNS) {
        float2 ml[U];
        float4 x[U][2];
#pragma unroll
        for (int u = 0; u < U; u++) {   // (all loads on their way; past the end: the last one again, left out)
            const uint64_t row = row_of(min(i0 + u, segments - 1));
            ml[u] = *reinterpret_cast<const float2 *>(p.ml + row * 2);
            const float4 *src = reinterpret_cast<const float4 *>(p.acc + (row & ~31ull) * D) + piece * 64 + (row & 31);
            x[u][0] = src[0];    // columns 8 piece .. + 3
            x[u][1] = src[32];   // columns 8 piece + 4 .. + 7
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (i0 + u < segments) {
                const float f[8] = {x[u][0].x, x[u][0].y, x[u][0].z, x[u][0].w, x[u][1].x, x[u][1].y, x[u][1].z, x[u][1].w};
                join(ml[u].x, ml[u].y, f);
            }
        }
    }
    if (shared) {
        if (turn != 0) {
            part[turn - 1][8][in_set] = m_all;
            part[turn - 1][9][in_set] = l;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                part[turn - 1][e][in_set] = o[e];
            }
        }
        __syncthreads();
        if (turn != 0) {
            return;
        }
#pragma unroll
        for (int u = 0; u < TURNS - 1; u++) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                f[e] = part[u][e][in_set];
            }
            join(part[u][8][in_set], part[u][9][in_set], f);
        }
    }
    if (m >= m_rows) {
        return;
    }
    const float inv = l > 0.f ? 1.0f / l : 0.f;
    const float scale = l != l ? l : inv;
    uint4 w;
    w.x = T::pack(o[0] * scale, o[1] * scale);
    w.y = T::pack(o[2] * scale, o[3] * scale);
    w.z = T::pack(o[4] * scale, o[5] * scale);
    w.w = T::pack(o[6] * scale, o[7] * scale);
    const uint64_t head = static_cast<uint64_t>(start + m / G) * p.n_heads + (WIDE ? kvh / 2 : kvh) * G + m % G;
    *reinterpret_cast<uint4 *>(p.out + (WIDE ? head * 2 + kvh % 2 : head) * D + piece * 8) = w;
}

// The kv heads of a workgroup: as many as divide the model's and leave it the rows of a typical M tile (twice the average of
// the batch, no more than the mask has nodes for). Two, one: 64 trees of 32 over 8192 positions 538 / 606 us, 16 ragged ones 58 /
// 63, int8 65 / 70, head_dim 64 25 / 28 (a few calls, not warm); trees of 60 nodes, whose rows need both M tiles, 126 / 128.
uint32_t heads_of(uint32_t total_tokens, uint32_t group, uint32_t n_kv_heads, uint32_t batch, uint32_t mask_words)
{
    const uint64_t rows = std::min<uint64_t>(2ull * total_tokens / batch, 32ull * mask_words) * group;
    return n_kv_heads % 2 == 0 && rows < 2 * kRows<2> ? 2u : 1u;
}

struct StreamPlan {
    uint32_t nh, groups, tiles, slots;
    size_t bytes;
};
StreamPlan plan_of(uint32_t total_tokens, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t batch, uint32_t block_size,
                   uint32_t max_num_block, uint32_t nh)
{
    StreamPlan s;
    const uint32_t G = n_heads / n_kv_heads, rows = 32 * kWaves / nh;
    s.nh = nh;
    s.groups = n_kv_heads / nh;
    s.tiles = static_cast<uint32_t>(static_cast<uint64_t>(total_tokens) * G / rows) + batch;
    // chunks: one per workgroup, more when a chunk's blocks would not fit the table
    const uint64_t sp = kHalf / 256 / nh, per = std::max<uint64_t>(1, (kTblCap - 2) * static_cast<uint64_t>(block_size) / sp);
    const uint64_t steps = s.tiles * ((static_cast<uint64_t>(max_num_block) * block_size + sp - 1) / sp);
    s.slots = static_cast<uint32_t>(2 * std::max<uint64_t>(std::max(1u, kComputeUnits / s.groups), steps / per + 1));
    s.bytes = s.tiles * sizeof(int4) + static_cast<size_t>(s.groups) * s.slots * nh * rows * (head_dim + 2) * sizeof(float);
    return s;
}

}  // namespace

// head_dim 64, 128 or 256 (16-bit caches); a copy's positions share a block (rows of 256 bytes: four of them; short rows have an address per lane); every
// block that a step can reach has its table entry in LDS; the kernel divides by the block size with its magic only (not blocks of 1)
bool tree_stream_supported(uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t block_size, uint32_t batch,
                           uint32_t max_num_block, int kv_dtype)
{
    return (head_dim == 128 || head_dim == 64 || (head_dim == 256 && kv_dtype == XLITE_HIP_KV_SAME)) && n_kv_heads > 0 && n_heads % n_kv_heads == 0 &&
           (block_size % 4 == 0 || head_dim == 64 || kv_dtype != XLITE_HIP_KV_SAME) &&
           batch <= kSeqCap && block_magic(block_size, static_cast<uint64_t>(max_num_block) * block_size) != 0;
}

size_t tree_stream_workspace_bytes(uint32_t total_tokens, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t batch,
                                   uint32_t block_size, uint32_t max_num_block)
{
    if (head_dim == 256) {   // as twice the heads of 128
        return plan_of(total_tokens, 2 * n_heads, 2 * n_kv_heads, 128, batch, block_size, max_num_block, 2).bytes;
    }
    size_t need = 0;   // whatever heads_of will say
    for (uint32_t nh : {1u, 2u}) {
        if (n_kv_heads % nh == 0) {
            need = std::max(need, plan_of(total_tokens, n_heads, n_kv_heads, head_dim, batch, block_size, max_num_block, nh).bytes);
        }
    }
    return need;
}

int launch_tree_stream(hipStream_t stream, const AttentionArgs &a)
{
    const bool wide = a.head_dim == 256;
    const uint32_t split = wide ? 2u : 1u, n_kv_heads = split * a.n_kv_heads, head_dim = a.head_dim / split;   // as they lie in memory
    const StreamPlan plan = plan_of(a.total_tokens, split * a.n_heads, n_kv_heads, head_dim, a.batch, a.block_size, a.max_num_block,
                                    wide ? 2u : heads_of(a.total_tokens, a.n_heads / a.n_kv_heads, a.n_kv_heads, a.batch, a.mask_words));
    if (a.workspace == nullptr || a.workspace_bytes < plan.bytes) {
        return fail(XLITE_HIP_ENOSPC, __func__, "workspace too small: need " + std::to_string(plan.bytes) + " bytes, have " +
                                                    std::to_string(a.workspace == nullptr ? 0 : a.workspace_bytes));
    }
    StreamParams p{};
    p.q = static_cast<const uint16_t *>(a.qkv);
    p.k_cache = static_cast<const unsigned char *>(a.k_cache);
    p.v_cache = static_cast<const unsigned char *>(a.v_cache);
    p.k_scale = a.k_scale;
    p.v_scale = a.v_scale;
    p.out = static_cast<uint16_t *>(a.output);
    p.tree_mask = a.tree_mask;
    p.query_start_loc = a.query_start_loc;
    p.lens = a.lens;
    p.cached_lens = a.cached_lens;
    p.block_tables = a.block_tables;
    p.q_tok_stride = (a.n_heads + 2 * a.n_kv_heads) * a.head_dim;
    p.n_heads = a.n_heads;
    p.n_kv_heads = n_kv_heads;
    p.group = a.n_heads / a.n_kv_heads;
    p.batch = a.batch;
    p.block_size = a.block_size;
    p.block_magic = block_magic(a.block_size, static_cast<uint64_t>(a.max_num_block) * a.block_size);
    p.max_num_block = a.max_num_block;
    p.mask_words = a.mask_words;
    p.slots = plan.slots;
    p.meta = static_cast<int4 *>(a.workspace);
    p.acc = reinterpret_cast<float *>(p.meta + plan.tiles);
    p.ml = p.acc + static_cast<uint64_t>(plan.groups) * plan.slots * 32 * kWaves * head_dim;
    const dim3 grid(std::max(1u, kComputeUnits / plan.groups), plan.groups), merge_grid(plan.tiles, n_kv_heads, 32 * kWaves / plan.nh / 16);
    auto launch = [&](auto t, auto n, auto kvf, auto io, auto d, auto w) -> int {
        using T = decltype(t);
        using TIO = decltype(io);
        constexpr int NH = decltype(n)::value, KVF = decltype(kvf)::value, D = decltype(d)::value;
        constexpr bool WIDE = decltype(w)::value;
        auto kernel = tree_stream_kernel<T, NH, KVF, TIO, D, WIDE>;
        const size_t lds = kStageBytes<KVF != XLITE_HIP_KV_SAME || D == 64> + (kTblCap + kMaskCap + a.batch + 1) * sizeof(uint32_t);
        if (const int rc = ensure_dynamic_lds(reinterpret_cast<const void *>(kernel), lds)) {
            return rc;
        }
        kernel<<<grid, kThreads, lds, stream>>>(p);
        XL_LAUNCH_CHECK();
        // few sequences: their tiles have a segment in (nearly) every workgroup; 250 segments of one tile took 64 us one set
        // after the other. Many: five segments are joined as fast by one set (8 us for 16 sequences, 10 with four sets)
        constexpr int SETS = 512 / D;
        if (grid.x >= 16 * a.batch) {
            tree_merge_kernel<TIO, NH, D, SETS, WIDE><<<merge_grid, 2 * D * SETS, 0, stream>>>(p);
        } else {
            tree_merge_kernel<TIO, NH, D, 1, WIDE><<<merge_grid, 2 * D, 0, stream>>>(p);
        }
        XL_LAUNCH_CHECK();
        return XLITE_HIP_OK;
    };
    auto with_heads = [&](auto t, auto kvf, auto io, auto d) -> int {
        return plan.nh == 2 ? launch(t, std::integral_constant<int, 2>{}, kvf, io, d, std::false_type{})
                            : launch(t, std::integral_constant<int, 1>{}, kvf, io, d, std::false_type{});
    };
    using D64 = std::integral_constant<int, 64>;
    using D128 = std::integral_constant<int, 128>;
    auto with_dim = [&](auto t, auto kvf, auto io) -> int {
        return a.head_dim == 128 ? with_heads(t, kvf, io, D128{}) : with_heads(t, kvf, io, D64{});
    };
    auto with_bytes = [&](auto kvf) -> int { return a.dtype == XLITE_HIP_BF16 ? with_dim(FP16{}, kvf, BF16{}) : with_dim(FP16{}, kvf, FP16{}); };
    switch (a.kv_dtype) {
    case XLITE_HIP_KV_INT8: return with_bytes(std::integral_constant<int, XLITE_HIP_KV_INT8>{});
    case XLITE_HIP_KV_FP8: return with_bytes(std::integral_constant<int, XLITE_HIP_KV_FP8>{});
    default: break;
    }
    using Same = std::integral_constant<int, XLITE_HIP_KV_SAME>;
    if (wide) {
        using Two = std::integral_constant<int, 2>;
        return a.dtype == XLITE_HIP_BF16 ? launch(BF16{}, Two{}, Same{}, BF16{}, D128{}, std::true_type{})
                                         : launch(FP16{}, Two{}, Same{}, FP16{}, D128{}, std::true_type{});
    }
    return a.dtype == XLITE_HIP_BF16 ? with_dim(BF16{}, Same{}, BF16{}) : with_dim(FP16{}, Same{}, FP16{});
}

}  // namespace xlite
