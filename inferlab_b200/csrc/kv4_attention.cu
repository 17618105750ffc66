// kv4_attention.cu - attention over a packed 4-bit pool (kv4.cuh): one decode
// step, and several query tokens per sequence. Many rows per kv-head have kernels
// of their own (kv4_prefill_tc.cuh, kv4_rows.cuh); plan_kv4 chooses.
//
// For a query q and the keys it sees, s_t = q . k_t / sqrt(D), p_t = exp(s_t -
// m), out = sum p_t v_t / sum p_t in one pass over the tokens with a running
// maximum m. With k = (c - 8) scale + zero per 64 dims,
//   s   = sum_groups [ scale (q . c) + (zero - 8 scale) (q . 1) ]
//   out = sum_t p_t scale_t (c_t - 8) + sum_t p_t zero_t,
// so both products run on the codes, which mma.sync takes as small exact
// numbers, and the pairs meet only scores and weights: 4 numbers per 16 tokens
// and lane instead of one per value.
//   scores: K codes as f16. A nibble in bits 0-3 of a half is the f16 subnormal
//     c 2^-24, in bits 4-7 it is c 2^-20, so a mask is the whole conversion; q
//     is scaled by a power of two per row (exact) into f16's range, and by 2^-4
//     where it meets the latter.
//   output: V codes as such f16 numbers less 8 of their unit, one mask and one
//     subtraction for two (each unit belongs to rows of the result, which are
//     scaled at the end), and
//     the weights p scale as f16, in two parts (22 bits together) for fp32
//     results. f16's range is kept by what m is: not the largest score but the
//     largest p scale, kept between 2^10 and 2^15, so that the first part loses
//     bits only 24 octaves below it and the second 13; l and the zero sums are
//     in the same unit.
// The mma computes S^T = K Q^T and O^T = V^T P^T: 16 tokens or dims by 8 query
// columns. P^T's operand layout is S^T's result transposed (movmatrix).
//
// What bounds it: (D + D / 8) bytes a token and kv-head from HBM (144 at D = 128,
// 23 bytes a clock and SM), and behind them the instructions of four warps a
// scheduler, which use 67% of its slots and mostly wait on each other's fixed
// latencies: 64 sequences of 4096 to 32768 tokens x 8 kv-heads, 4 queries each,
// 1489 MB in 280 to 327 us with the card and its clock under load (5.3 to 4.6
// TB/s). One CTA of four warps per (sequence, kv-head, 8 columns, split); every
// warp streams its own 16-token tiles through a ring in shared memory, so that
// the warps never wait for each other before the merge. The copies are 16-byte
// cp.async by all lanes: five instructions a tile, where a bulk copy by one lane
// with its barrier took ~40 issue slots of ~430.
#include "common.cuh"
#include "internal.cuh"
#include "kv4.cuh"
#include "pool.cuh"

#include "../../include/inferlab_attention.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

namespace ilb {
namespace {

constexpr int kWarps = 4;
constexpr int kRing = 3;                // steps in a warp's ring
constexpr int kStep = 2;               // tiles a warp takes at once
constexpr float kHeadroom = 10.0f;     // log2: the largest scaled weight starts at 2^10 (below)
constexpr float kNoScore = -3.0e38f;   // running maximum before any key
constexpr std::uint32_t kMaxSplits = 256;
// The split counters lie at the front of a workspace and are zero between
// launches; behind them are the partials of whatever batch ran last. So the
// region is the same for all batches. More units than this fill the GPU many
// times over and are not split.
constexpr std::uint32_t kMaxSplitUnits = 16384;
constexpr std::uint32_t kMaxSplitCtas = 32768;  // of split batches, where the planner chooses

struct Kv4Params {
    const unsigned char* arena;
    std::uint64_t num_blocks;
    std::uint32_t kv_heads, q_heads, group, tiles_per_block;
    const void* queries;
    void* out;
    const std::int32_t* tables;
    std::uint32_t max_blocks;
    int max_context;
    const std::int32_t* context_lens;  // decode; null: segments
    const std::int32_t* starts;
    const std::int32_t* counts;
    const std::int32_t* offsets;
    std::uint32_t num_seqs;
    std::uint32_t max_count;           // query tokens a sequence may have
    long long total_queries;
    std::uint32_t column_tiles, max_splits;
    std::uint32_t per_seq;             // kv-heads x column (or row) tiles
    bool by_length;                    // longest contexts first
    int tiles_per_split;
    float scale_log2;
    std::uint32_t* ws_count;  // [unit]
    float* ws_part;           // [unit][split]: o [columns][D], then (m, l) per column, padded to [columns][D + 4]
    std::uint32_t* error_word;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], std::uint32_t a0, std::uint32_t a1,
                                        std::uint32_t a2, std::uint32_t a3, std::uint32_t b0,
                                        std::uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same onto zero.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], std::uint32_t a0, std::uint32_t a1,
                                              std::uint32_t a2, std::uint32_t a3, std::uint32_t b0,
                                              std::uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ std::uint32_t transpose8(std::uint32_t x) {
    std::uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// Two masked codes c 2^-24 (low nibbles) or c 2^-20 (high ones) as f16, less 8
// of that unit: exact, subnormal or not.
__device__ __forceinline__ std::uint32_t centred_low(std::uint32_t x) {
    x &= 0x000f000fu;
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x0008)));
    return *reinterpret_cast<const std::uint32_t*>(&v);
}
__device__ __forceinline__ std::uint32_t centred_high(std::uint32_t x) {
    x &= 0x00f000f0u;
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x0080)));
    return *reinterpret_cast<const std::uint32_t*>(&v);
}
__device__ __forceinline__ std::uint32_t f16_pair(float low, float high) {
    const __half2 v = __floats2half2_rn(low, high);
    return *reinterpret_cast<const std::uint32_t*>(&v);
}
// The (scale, zero) pairs of N neighbouring groups.
__device__ __forceinline__ void load_pairs(const unsigned char* at, float2 (&pairs)[1]) {
    pairs[0] = __half22float2(*reinterpret_cast<const __half2*>(at));
}
__device__ __forceinline__ void load_pairs(const unsigned char* at, float2 (&pairs)[2]) {
    const uint2 raw = *reinterpret_cast<const uint2*>(at);
    pairs[0] = __half22float2(*reinterpret_cast<const __half2*>(&raw.x));
    pairs[1] = __half22float2(*reinterpret_cast<const __half2*>(&raw.y));
}
// What m may be for a score and the log2 of what its weight is multiplied by:
// `kHeadroom` below their sum, rounded up and never above the score. From 2^24
// on, fp32 scores are so far apart that the headroom itself is rounded: rounded
// down, m would let 2^(score - m) times that factor leave f16's range (scores
// around 2^28); rounded up it may be lost, and the weight is then 1 and what is
// kept as f16 the factor itself.
__device__ __forceinline__ float score_with_room(float score, float factor_log2) {
    return __fadd_ru(score, fminf(factor_log2 - kHeadroom, 0.0f));
}
// Token slot (0..7) that sits in row r of an 8-token mma half: r = 2t is token
// t, r = 2t + 1 token 7 - t. Rows 2t of all t (what four lanes read of V at
// once) and rows r of neighbouring r (K) then fall on different banks.
__device__ __forceinline__ int slot_of_row(int r) { return r & 1 ? 7 - (r >> 1) : r >> 1; }

// What a CTA works on: a split of a sequence's keys, and which of its kv-heads
// and tiles. By length (run_kv4 says for which batches), sequences come in the
// order of their contexts, which the device knows, all of a long one's CTAs before
// a shorter one's: the short ones fill what the long ones leave. Otherwise the last splits come first, which only long contexts have;
// row tiles (kRowTiles: rest = tile x kv-heads + kv-head) then before the
// sequences, those with the most keys first (8 prompts of 1 to 1024 tokens: 66
// us, 82 sequence by sequence).
struct Work {
    std::uint32_t seq, split, rest;
};
template <bool kRowTiles>
__device__ __forceinline__ Work work_of(const Kv4Params& p) {
    Work w;
    if (!p.by_length) {
        const std::uint32_t units = p.num_seqs * p.per_seq, unit = blockIdx.x % units;
        w.split = p.max_splits - 1 - blockIdx.x / units;
        if constexpr (kRowTiles) {
            const std::uint32_t pairs = p.num_seqs * p.kv_heads, pair = unit % pairs;
            w.seq = pair / p.kv_heads;
            w.rest = unit / pairs * p.kv_heads + pair % p.kv_heads;
        } else {
            w.seq = unit / p.per_seq;
            w.rest = unit % p.per_seq;
        }
        return w;
    }
    const int lane = threadIdx.x & 31;
    auto length_of = [&](std::uint32_t seq) -> std::uint32_t {  // 1 more than the context; 0 for no sequence
        if (seq >= p.num_seqs) return 0;
        return 1 + (p.context_lens != nullptr ? static_cast<std::uint32_t>(p.context_lens[seq])
                                              : static_cast<std::uint32_t>(p.starts[seq]) + static_cast<std::uint32_t>(p.counts[seq]));
    };
    // Ranks of sequences lane and 32 + lane; of equal ones the first comes first.
    const std::uint32_t low = length_of(lane), high = length_of(32 + lane);
    std::uint32_t low_rank = 0, high_rank = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const std::uint32_t other = __shfl_sync(0xffffffffu, low, i);
        low_rank += other > low || (other == low && i < lane);
        high_rank += other >= high;
    }
    if (p.num_seqs > 32) {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const std::uint32_t other = __shfl_sync(0xffffffffu, high, i);
            low_rank += other > low;
            high_rank += other > high || (other == high && i < lane);
        }
    }
    const std::uint32_t each = p.per_seq * p.max_splits, at = blockIdx.x % each;
    const std::uint32_t rank = blockIdx.x / each;
    const std::uint32_t in_low = __ballot_sync(0xffffffffu, low_rank == rank), in_high = __ballot_sync(0xffffffffu, high_rank == rank);
    w.seq = in_low != 0 ? __ffs(in_low) - 1 : 31 + __ffs(in_high);
    w.split = at / p.per_seq;
    w.rest = at % p.per_seq;
    return w;
}

// Whether this CTA is the last of `splits` to come here; what the others wrote
// before is then visible. Returns the counter to zero.
__device__ __forceinline__ bool last_of(std::uint32_t* counter, int splits, std::uint32_t& ticket) {
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        ticket = atomicAdd(counter, 1u);
        if (ticket == static_cast<std::uint32_t>(splits) - 1) *counter = 0;
        __threadfence();
    }
    __syncthreads();
    return ticket == static_cast<std::uint32_t>(splits) - 1;
}

// Four dims (the i-th of a part) of a row merged over the splits in their order,
// one round of loads for each kRound of them. A part is kPart floats: o, then
// from kMl on (m, l) per row.
template <int kPart, int kMl>
__device__ __forceinline__ float4 merge_parts(const float* parts, int splits, int row, int i, bool& ok) {
    constexpr int kRound = 8;
    float top = kNoScore, sum = 0.0f;
    float4 total = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k0 = 0; k0 < splits; k0 += kRound) {
        float2 ml[kRound];
        float4 x[kRound];
#pragma unroll
        for (int k = 0; k < kRound; ++k) {
            const float* at = parts + static_cast<std::size_t>(min(k0 + k, splits - 1)) * kPart;
            ml[k] = __ldcg(reinterpret_cast<const float2*>(at + kMl + 2 * row));
            x[k] = __ldcg(reinterpret_cast<const float4*>(at) + i);
        }
        float next = top;
#pragma unroll
        for (int k = 0; k < kRound; ++k) next = fmaxf(next, ml[k].x);
        const float kept = ex2_ftz(top - next);
        sum *= kept;
        total.x *= kept, total.y *= kept, total.z *= kept, total.w *= kept;
        top = next;
#pragma unroll
        for (int k = 0; k < kRound; ++k) {
            const float w = k0 + k < splits ? ex2_ftz(ml[k].x - top) : 0.0f;
            sum = fmaf(w, ml[k].y, sum);
            total.x = fmaf(w, x[k].x, total.x);
            total.y = fmaf(w, x[k].y, total.y);
            total.z = fmaf(w, x[k].z, total.z);
            total.w = fmaf(w, x[k].w, total.w);
        }
    }
    ok = isfinite(sum) && sum > 0.0f;
    const float inv = ok ? 1.0f / sum : 0.0f;
    return make_float4(total.x * inv, total.y * inv, total.z * inv, total.w * inv);
}

template <typename QT>
__device__ __forceinline__ void store_row4(QT* out, float4 x) {
    if constexpr (sizeof(QT) == 4) {
        *reinterpret_cast<float4*>(out) = x;
    } else {
        QT v[4] = {Storage<QT>::from_float(x.x), Storage<QT>::from_float(x.y), Storage<QT>::from_float(x.z),
                   Storage<QT>::from_float(x.w)};
        *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(v);
    }
}

// Up to 8 live query columns, or (kFour) up to 4 that stand twice, so that
// columns 4-7 carry something else of the same queries:
//   fp32 queries: the second part of the weights (8 columns: a second product);
//   16-bit queries, whose outputs are rounded to 2^-12 or 2^-9 anyway, take the
//   weights in one f16 part (2^-12 each, before they average out), and with
//   D = 128 columns 4-7 the weights scaled for dims 64-127 instead of 0-63: a
//   lane then has one value pair per token, and the columns of the other half
//   of the dims are not used.
template <typename RowT, typename QT, int D, bool kFour>
__global__ void __launch_bounds__(kWarps * 32, 4) kv4_attention_kernel(const Kv4Params p) {
    constexpr int kTile = kv4::tile_bytes(D);
    constexpr int kGroups = D / kv4::kGroup;
    constexpr int kWords = D / 32;  // key words of a lane and token
    constexpr int kMt = D / 16;     // 16-dim tiles of the output
    constexpr int kCols = kFour ? 4 : 8;
    constexpr bool kTwoParts = std::is_same<QT, float>::value;
    constexpr bool kByGroup = kFour && !kTwoParts && kGroups == 2;
    constexpr int kPairs = kByGroup ? 1 : kGroups;  // value pairs of a lane and token
    constexpr int kStepBytes = kStep * kTile;
    constexpr int kRegion = kRing * kStepBytes;  // a warp's ring, and later its state
    static_assert(kCols * (D + 2) * 4 <= kRegion, "a warp's state must fit its ring");
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ std::uint32_t ticket;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t4 = lane & 3;
    const Work work = work_of<false>(p);
    const std::uint32_t seq = work.seq, split = work.split;
    const std::uint32_t column_tile = work.rest % p.column_tiles, kv_head = work.rest / p.column_tiles;
    const std::uint32_t unit = seq * p.per_seq + work.rest;
    const int b0 = static_cast<int>(split) * p.tiles_per_split;

    // Block ids of the split's first tiles are asked for at once, beside the
    // context length (an entry behind the sequence's last block is not used).
    // The warp's tiles: kStep neighbours, then kStep past the other warps'.
    // Lane i has tile i of the first kAhead, then tile kAhead + 32 k + i.
    constexpr int kAhead = kRing * kStep;
    const std::int32_t* table = p.tables + static_cast<std::size_t>(seq) * p.max_blocks;
    auto tile_of = [&](int i) { return static_cast<std::uint32_t>(b0 + kStep * (warp + kWarps * (i / kStep)) + i % kStep); };
    auto block_of = [&](int i) { return table[min(tile_of(i) / p.tiles_per_block, p.max_blocks - 1)]; };
    const std::int32_t first_blocks = lane < kAhead ? block_of(lane) : 0;
    std::int32_t next_blocks = block_of(kAhead + lane);

    // ---- what this CTA works on: columns r0 .. r0 + live - 1 of the sequence's
    // count * group query rows (token-major), keys 0 .. longest - 1.
    std::uint32_t start, count, offset;
    bool valid;
    if (p.context_lens != nullptr) {
        const std::int32_t ctx = p.context_lens[seq];
        valid = ctx >= 0 && ctx <= p.max_context;
        start = static_cast<std::uint32_t>(ctx) - 1;
        count = 1;
        offset = seq;
        if (!valid && split == 0 && threadIdx.x == 0) flag_error(p.error_word, kErrContext);
    } else {
        const std::int32_t s = p.starts[seq], c = p.counts[seq], o = p.offsets[seq];
        start = static_cast<std::uint32_t>(s);
        count = static_cast<std::uint32_t>(c);
        offset = static_cast<std::uint32_t>(o);
        valid = s >= 0 && c >= 0 && static_cast<long long>(s) + c <= p.max_context;
        const bool rows_ok = c >= 0 && count <= p.max_count && o >= 0 && static_cast<long long>(o) + c <= p.total_queries;
        if (!(valid && rows_ok) && split == 0 && threadIdx.x == 0) flag_error(p.error_word, kErrSegment);
        if (!rows_ok) return;
    }
    const std::uint32_t r0 = column_tile * kCols;
    if (r0 >= count * p.group) return;
    const int live = static_cast<int>(min(static_cast<std::uint32_t>(kCols), count * p.group - r0));
    auto row_of = [&](int col) -> std::size_t {  // the row of queries / out of a live column
        const std::uint32_t token = (r0 + col) / p.group;
        return static_cast<std::size_t>(offset + token) * p.q_heads + kv_head * p.group + (r0 + col - token * p.group);
    };
    const int longest = valid ? static_cast<int>(start + (r0 + live - 1) / p.group + 1) : 0;
    if (longest == 0) {  // no sequence, or a bad one: zero rows
        if (split == 0) {
            for (int i = threadIdx.x; i < live * D; i += blockDim.x) {
                static_cast<QT*>(p.out)[row_of(i / D) * D + i % D] = Storage<QT>::from_float(0.0f);
            }
        }
        return;
    }
    const int tiles = (longest + kv4::kTileTokens - 1) / kv4::kTileTokens;
    const int splits = (tiles + p.tiles_per_split - 1) / p.tiles_per_split;
    if (static_cast<int>(split) >= splits) return;
    const int nb = min(tiles - b0, p.tiles_per_split);
    const int mine = [&] {
        const int whole = nb / (kStep * kWarps) * kStep, rest = nb % (kStep * kWarps) - kStep * warp;
        return whole + min(max(rest, 0), kStep);
    }();

    // ---- the ring: 16-byte asynchronous copies by all lanes, one group a step.
    unsigned char* ring = smem + warp * kRegion;
    auto tile_address = [&](int i, std::int32_t block) -> std::uint64_t {
        if (i >= mine) return 0;
        if (block < 0 || static_cast<std::uint64_t>(block) >= p.num_blocks) {
            flag_error(p.error_word, kErrBadBlock);
            block = 0;  // never dereferenced outside the pool
        }
        const std::uint64_t at = (static_cast<std::uint64_t>(block) * p.kv_heads + kv_head) * p.tiles_per_block + tile_of(i) % p.tiles_per_block;
        return reinterpret_cast<std::uint64_t>(p.arena) + at * kTile;
    };
    std::uint64_t addresses = lane < kAhead ? tile_address(lane, first_blocks) : 0;
    const std::uint32_t ring_at = smem_u32(ring) + lane * 16;
    auto fetch = [&](std::uint32_t to, std::uint64_t from) {  // one tile
        const unsigned char* src = reinterpret_cast<const unsigned char*>(from) + lane * 16;
#pragma unroll
        for (int c = 0; c < kTile; c += 512) {
            if (c + 512 <= kTile || lane * 16 < kTile - c) cp_async16(to + c, src + c);
        }
    };
    // ---- queries as the B operand: lane holds column g, dims 32 w + 8 t4 + 0..7.
    std::uint32_t qf[kWords][4];
    float q_sum[kGroups][2], factor[2];  // of this lane's result columns 2 t4, 2 t4 + 1
    int limit[2];                        // keys they see
    {
        const int col = kFour ? g & 3 : g;
        float x[kWords][8];
        float most = 0.0f;
        bool bad = false;
        // Asked for before the tiles, which would keep them waiting.
        const QT* row = static_cast<const QT*>(p.queries) + row_of(min(col, live - 1)) * D + 8 * t4;
        constexpr int kPer = 16 / sizeof(QT);
        uint4 raw[kWords][8 / kPer];
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
#pragma unroll
            for (int c = 0; c < 8 / kPer; ++c) raw[w][c] = reinterpret_cast<const uint4*>(row + 32 * w)[c];
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const std::uint64_t from = __shfl_sync(0xffffffffu, addresses, i);
            if (i < mine) fetch(ring_at + i * kTile, from);
            if (i % kStep == kStep - 1) cp_async_commit();
        }
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
#pragma unroll
            for (int c = 0; c < 8 / kPer; ++c) widen16(raw[w][c], &x[w][c * kPer], QT{});
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[w][i] = col < live ? Storage<RowT>::to_float(Storage<RowT>::from_float(x[w][i])) : 0.0f;
                bad |= !isfinite(x[w][i]);
                most = fmaxf(most, fabsf(x[w][i]));
            }
        }
        if (bad) flag_error(p.error_word, kErrNonFinite);
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // A power of two brings the row's largest number to [2^14, 2^15).
        const int exponent = max(15, static_cast<int>(__float_as_uint(most) >> 23));
        const float up = most > 0.0f ? __uint_as_float(static_cast<std::uint32_t>(min(254, 268 - exponent)) << 23) : 1.0f;
        float sums[kGroups];
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
            if (w % 2 == 0) sums[w / 2] = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[w][i] *= up;
                sums[w / 2] += x[w][i];
            }
            qf[w][0] = f16_pair(x[w][0], x[w][4]);
            qf[w][1] = f16_pair(x[w][2], x[w][6]);
            qf[w][2] = f16_pair(x[w][1] * 0.0625f, x[w][5] * 0.0625f);
            qf[w][3] = f16_pair(x[w][3] * 0.0625f, x[w][7] * 0.0625f);
        }
        // 2^24 undoes the subnormal codes' 2^-24; q_sum carries that factor too.
        const float down = fminf(p.scale_log2 * 16777216.0f / up, 3.0e38f);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int from = (2 * t4 + c) * 4;
            factor[c] = __shfl_sync(0xffffffffu, down, from);
            const int cc = kFour ? (2 * t4 + c) & 3 : 2 * t4 + c;
            limit[c] = cc < live ? static_cast<int>(start + (r0 + cc) / p.group + 1) : 0;
        }
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
            float s = sums[k];
            s += __shfl_xor_sync(0xffffffffu, s, 1);
            s += __shfl_xor_sync(0xffffffffu, s, 2);
            s *= 5.9604644775390625e-08f;
#pragma unroll
            for (int c = 0; c < 2; ++c) q_sum[k][c] = __shfl_sync(0xffffffffu, s, (2 * t4 + c) * 4);
        }
    }
    const int shortest = static_cast<int>(start + r0 / p.group + 1);  // keys every live column sees

    float m[2] = {kNoScore, kNoScore}, l[2] = {0.0f, 0.0f};
    float z[kPairs][2];
    float o[kMt][4];
#pragma unroll
    for (int k = 0; k < kPairs; ++k) z[k][0] = z[k][1] = 0.0f;
#pragma unroll
    for (int i = 0; i < kMt; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    const int slot = slot_of_row(g);
    const std::uint32_t second_part = kFour && t4 >= 2 ? 0xffffffffu : 0u;
    const int key_at = slot * (D / 2) + t4 * (D / 8);
    const int pair_key = kv4::pair_at(D, slot, 0, 0), pair_value = kv4::pair_at(D, slot, kByGroup ? t4 >> 1 : 0, 1);
    const int value_a = kv4::value_word(D, t4, g), value_b = kv4::value_word(D, 7 - t4, g);
    const int end = min(longest, (b0 + nb) * kv4::kTileTokens);
    const int clear = min(shortest, end);  // keys below it are this split's and every live column's

    // Per step: scores of the next one beside the output product of this one
    // (independent work for the scheduler), then the next one's weights.
    float s[kStep][4];  // (token half, column): scores in log2
    float2 vp[kStep][2][kPairs];
    std::uint32_t pf[kStep][kPairs][2], pf2[kStep][kPairs][2];
    auto scores = [&](const unsigned char* base) {
        // S^T: rows are tokens slot, slot + 8; per group of 64 dims.
#pragma unroll
        for (int u = 0; u < kStep; ++u) {
            const unsigned char* tile = base + u * kTile;
            float acc[kGroups][4];
            std::uint32_t k0[kWords], k1[kWords];
            if constexpr (D == 128) {
                const uint4 a = *reinterpret_cast<const uint4*>(tile + key_at);
                const uint4 b = *reinterpret_cast<const uint4*>(tile + key_at + 8 * (D / 2));
                k0[0] = a.x, k0[1] = a.y, k0[2] = a.z, k0[3] = a.w;
                k1[0] = b.x, k1[1] = b.y, k1[2] = b.z, k1[3] = b.w;
            } else {
                const uint2 a = *reinterpret_cast<const uint2*>(tile + key_at);
                const uint2 b = *reinterpret_cast<const uint2*>(tile + key_at + 8 * (D / 2));
                k0[0] = a.x, k0[1] = a.y, k1[0] = b.x, k1[1] = b.y;
            }
#pragma unroll
            for (int w = 0; w < kWords; ++w) {
                const std::uint32_t h0 = k0[w] >> 8, h1 = k1[w] >> 8;
                if (w % 2 == 0) {
                    mma_f16_first(acc[w / 2], k0[w] & 0x000f000fu, k1[w] & 0x000f000fu, h0 & 0x000f000fu,
                                  h1 & 0x000f000fu, qf[w][0], qf[w][1]);
                } else {
                    mma_f16(acc[w / 2], k0[w] & 0x000f000fu, k1[w] & 0x000f000fu, h0 & 0x000f000fu, h1 & 0x000f000fu,
                            qf[w][0], qf[w][1]);
                }
                mma_f16(acc[w / 2], k0[w] & 0x00f000f0u, k1[w] & 0x00f000f0u, h0 & 0x00f000f0u, h1 & 0x00f000f0u,
                        qf[w][2], qf[w][3]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float2 kp[kGroups];
                load_pairs(tile + pair_key + 8 * h * kGroups * 4, kp);
#pragma unroll
                for (int k = 0; k < kGroups; ++k) {
                    const float rest = fmaf(-8.0f, kp[k].x, kp[k].y);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float& x = s[u][2 * h + c];
                        x = k == 0 ? rest * q_sum[k][c] : fmaf(rest, q_sum[k][c], x);
                        x = fmaf(kp[k].x, acc[k][2 * h + c], x);
                    }
                }
            }
            // Rounded before m is taken off: scores of 2^28 and more would
            // otherwise differ from their own maximum.
#pragma unroll
            for (int i = 0; i < 4; ++i) s[u][i] *= factor[i & 1];
        }
#pragma unroll
        for (int u = 0; u < kStep; ++u) {
#pragma unroll
            for (int h = 0; h < 2; ++h) load_pairs(base + u * kTile + pair_value + 8 * h * kGroups * 4, vp[u][h]);
        }
    };
    auto weights = [&](int first) {
        if (first + kStep * kv4::kTileTokens > clear) {
            // Slots behind the last key may hold anything; their pairs count as 0.
#pragma unroll
            for (int u = 0; u < kStep; ++u) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int token = first + kv4::kTileTokens * u + slot + 8 * h;
#pragma unroll
                    for (int c = 0; c < 2; ++c) s[u][2 * h + c] = token < min(limit[c], end) ? s[u][2 * h + c] : -INFINITY;
                    if (token >= end) {
#pragma unroll
                        for (int k = 0; k < kPairs; ++k) vp[u][h][k] = make_float2(0.0f, 0.0f);
                    }
                }
            }
        }
        // Weights 2^(s - m), and times the value scales, which must fit
        // f16: m moves when one outgrows 2^15 (or a weight 2^34, where scales
        // are tiny).
        float weight[kStep][4], scaled[kStep][2][kPairs][2];
        float most_weight = 0.0f, most_scaled = 0.0f;
        auto weigh = [&] {
#pragma unroll
            for (int u = 0; u < kStep; ++u) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        weight[u][2 * h + c] = ex2_ftz(s[u][2 * h + c] - m[c]);
#pragma unroll
                        for (int k = 0; k < kPairs; ++k) scaled[u][h][k][c] = weight[u][2 * h + c] * vp[u][h][k].x;
                    }
                    most_weight = fmax3(most_weight, weight[u][2 * h], weight[u][2 * h + 1]);
#pragma unroll
                    for (int k = 0; k < kPairs; ++k) most_scaled = fmax3(most_scaled, scaled[u][h][k][0], scaled[u][h][k][1]);
                }
            }
        };
        weigh();
        if (__any_sync(0xffffffffu, most_scaled > 32768.0f || most_weight > 17179869184.0f)) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float top = kNoScore;
#pragma unroll
                for (int u = 0; u < kStep; ++u) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float scale = 9.5367431640625e-07f;  // 2^-20
#pragma unroll
                        for (int k = 0; k < kPairs; ++k) scale = fmaxf(scale, vp[u][h][k].x);
                        top = fmaxf(top, score_with_room(s[u][2 * h + c], __log2f(scale)));
                    }
                }
                if constexpr (kFour) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));  // the column's twin
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                top = fmaxf(top, m[c]);
                const float alpha = ex2_ftz(m[c] - top);
                m[c] = top;
                l[c] *= alpha;
#pragma unroll
                for (int k = 0; k < kPairs; ++k) z[k][c] *= alpha;
#pragma unroll
                for (int i = 0; i < kMt; ++i) o[i][c] *= alpha, o[i][2 + c] *= alpha;
            }
            weigh();
        }

#pragma unroll
        for (int u = 0; u < kStep; ++u) {
            // P^T as the B operand, per value pair.
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                l[0] += weight[u][2 * h];
                l[1] += weight[u][2 * h + 1];
#pragma unroll
                for (int k = 0; k < kPairs; ++k) {
                    const float w0 = scaled[u][h][k][0], w1 = scaled[u][h][k][1];
                    z[k][0] = fmaf(weight[u][2 * h], vp[u][h][k].y, z[k][0]);
                    z[k][1] = fmaf(weight[u][2 * h + 1], vp[u][h][k].y, z[k][1]);
                    const std::uint32_t high = f16_pair(w0, w1);
                    if constexpr (kTwoParts) {
                        const std::uint32_t taken = kFour ? high & second_part : high;
                        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&taken));
                        const std::uint32_t left = f16_pair(w0 - t.x, w1 - t.y);
                        pf[u][k][h] = transpose8(kFour ? left : high);
                        if constexpr (!kFour) pf2[u][k][h] = transpose8(left);
                    } else {
                        pf[u][k][h] = transpose8(high);
                    }
                }
            }
        }
    };
    auto output = [&](const unsigned char* base) {
#pragma unroll
        for (int u = 0; u < kStep; ++u) {
            const unsigned char* tile = base + u * kTile;
            // O^T += V^T P^T: k index 2 t4 is token t4, 2 t4 + 1 token 7 - t4.
            std::uint32_t v[4][kGroups];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned char* at = tile + (i % 2 ? value_b : value_a) + i / 2 * 8 * (D / 2);
                if constexpr (D == 128) {
                    const uint2 x = *reinterpret_cast<const uint2*>(at);
                    v[i][0] = x.x, v[i][1] = x.y;
                } else {
                    v[i][0] = *reinterpret_cast<const std::uint32_t*>(at);
                }
            }
#pragma unroll
            for (int k = 0; k < kGroups; ++k) {
                constexpr int kLast = kPairs - 1;
                const std::uint32_t(&b)[2] = pf[u][k < kLast ? k : kLast];
                const std::uint32_t(&b2)[2] = pf2[u][k < kLast ? k : kLast];
#pragma unroll
                for (int half = 0; half < 2; ++half) {  // nibbles 0-3, 4-7: dims 8 g + 0..3, + 4..7
                    std::uint32_t x = __byte_perm(v[0][k], v[1][k], half ? 0x7632 : 0x5410);
                    std::uint32_t y = __byte_perm(v[2][k], v[3][k], half ? 0x7632 : 0x5410);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float (&d)[4] = o[4 * k + 2 * half + j];
                        const std::uint32_t a0 = centred_low(x), a1 = centred_high(x);
                        const std::uint32_t a2 = centred_low(y), a3 = centred_high(y);
                        mma_f16(d, a0, a1, a2, a3, b[0], b[1]);
                        if constexpr (kTwoParts && !kFour) mma_f16(d, a0, a1, a2, a3, b2[0], b2[1]);
                        x >>= 8, y >>= 8;
                    }
                }
            }
        }
    };
    int first = (b0 + kStep * warp) * kv4::kTileTokens;
    std::uint32_t in_ring = 0;
    int done = 0;
    for (; done < mine; done += kStep) {
        if ((done & 31) == 0) {
            addresses = tile_address(kAhead + done + lane, next_blocks);
            next_blocks = block_of(kAhead + done + 32 + lane);
        }
        cp_async_wait_group<kRing - 1>();
        __syncwarp();
        scores(ring + in_ring);
        weights(first);
        output(ring + in_ring);
        __syncwarp();  // this step's tiles are read
#pragma unroll
        for (int u = 0; u < kStep; ++u) {
            const std::uint64_t from = __shfl_sync(0xffffffffu, addresses, (done + u) & 31);
            if (kAhead + done + u < mine) fetch(ring_at + in_ring + u * kTile, from);
        }
        cp_async_commit();
        in_ring = in_ring + kStepBytes == kRegion ? 0 : in_ring + kStepBytes;
        first += kStep * kWarps * kv4::kTileTokens;
    }
    cp_async_wait_group<0>();
    __syncwarp();

    // ---- a warp's state into its ring: [column][D] output sums, then m and l.
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
            l[c] += __shfl_xor_sync(0xffffffffu, l[c], off);
#pragma unroll
            for (int k = 0; k < kPairs; ++k) z[k][c] += __shfl_xor_sync(0xffffffffu, z[k][c], off);
        }
    }
    float* state = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int i = 0; i < kMt; ++i) {
        if constexpr (kFour && kTwoParts) {  // both parts of the weights meet
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] += __shfl_xor_sync(0xffffffffu, o[i][e], 2);
        }
        const int dim = 64 * (i / 4) + 8 * g + 2 * (i % 4);
        const int pair = kPairs == 1 ? 0 : i / 4;
        const bool holds = kByGroup ? t4 >> 1 == i / 4 : !kFour || t4 < 2;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int col = (2 * t4 + c) & (kCols - 1);
            if (holds) {
                // Back from the codes' units: 2^24 in rows g, 2^20 in rows g + 8.
                *reinterpret_cast<float2*>(state + col * D + dim) =
                    make_float2(fmaf(o[i][c], 16777216.0f, z[pair][c]), fmaf(o[i][2 + c], 1048576.0f, z[pair][c]));
            }
        }
    }
    if (g == 0) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int col = 2 * t4 + c;
            if (col < kCols) state[kCols * D + 2 * col] = m[c], state[kCols * D + 2 * col + 1] = l[c];
        }
    }
    __syncthreads();
    auto state_of = [&](int w) { return reinterpret_cast<const float*>(smem + w * kRegion); };
    constexpr int kPart = kCols * (D + 4);  // a split's o [column][D], then m and l per column (padded)
    float* part = p.ws_part + (static_cast<std::size_t>(unit) * p.max_splits + split) * kPart;
    for (int i = threadIdx.x; i < live * D; i += blockDim.x) {
        const int col = i / D;
        float top = kNoScore, sum = 0.0f, total = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, state_of(w)[kCols * D + 2 * col]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float weight = ex2_ftz(state_of(w)[kCols * D + 2 * col] - top);
            sum = fmaf(weight, state_of(w)[kCols * D + 2 * col + 1], sum);
            total = fmaf(weight, state_of(w)[i], total);
        }
        if (splits == 1) {
            const bool ok = isfinite(sum) && sum > 0.0f;
            if (!ok) flag_error(p.error_word, kErrNormalizer);
            static_cast<QT*>(p.out)[row_of(col) * D + i % D] = Storage<QT>::from_float(ok ? total / sum : 0.0f);
        } else {
            part[i] = total;
            if (i % D == 0) part[kCols * D + 2 * col] = top, part[kCols * D + 2 * col + 1] = sum;
        }
    }
    if (splits == 1) return;

    // ---- the unit's last CTA merges the splits, every thread four dims.
    if (!last_of(p.ws_count + unit, splits, ticket)) return;
    const float* parts = p.ws_part + static_cast<std::size_t>(unit) * p.max_splits * kPart;
    for (int i = threadIdx.x; i < live * D / 4; i += blockDim.x) {
        const int col = i / (D / 4);
        bool ok;
        const float4 x = merge_parts<kPart, kCols * D>(parts, splits, col, i, ok);
        if (!ok) flag_error(p.error_word, kErrNormalizer);
        store_row4(static_cast<QT*>(p.out) + row_of(col) * D + 4 * i % D, x);
    }
}

}  // namespace
}  // namespace ilb

#include "kv4_rows.cuh"
#include "kv4_prefill_tc.cuh"

namespace ilb {
namespace {

// Columns a CTA works on, and how the keys are cut; or whole row tiles
// (kv4_rows.cuh).
struct Kv4Plan {
    std::uint32_t columns, column_tiles, max_splits;
    int tiles_per_split;
    std::size_t counter_bytes, part_bytes;
    enum { kColumns, kRows, kTensor } kind;
};

Kv4Plan plan_kv4(const InferlabCudaKvPool& p, std::uint32_t num_seqs, std::uint32_t q_heads,
                 std::uint32_t max_count, std::uint32_t max_context_len, std::uint32_t query_dtype) {
    Kv4Plan plan{};
    const std::uint64_t rows = static_cast<std::uint64_t>(q_heads / p.kv_heads) * max_count;
    if (rows > 0x7FFFFFFFull) throw std::runtime_error("4-bit attention batch is too large");
    // Many rows per kv-head share the widened codes. 16-bit queries from 64 rows
    // on: 64 segments on contexts of 1200 tokens take 180, 184 and 215 us with 48,
    // 64 and 128 rows on the tensor cores, 134, 175 and 342 in column tiles; 4 on
    // 8000 tokens 68, 71 and 81 against 65, 78 and 134. fp32 results need
    // weights in two parts and take the row kernel from 128 rows on, where its
    // tiles fill the GPU: 64 fresh prompts of 32 tokens 40 us against 108 in column
    // tiles, one prompt of 32 tokens (not filled) 13 against 10; where they meet,
    // 64 segments of 32 tokens on 1200, the row kernel is the slower one by 5%, 398
    // against 379.
    const bool tensor = query_dtype != kFp32;
    const std::uint64_t row_tile = tensor ? kTcRows : kRowTile, row_tiles = (rows + row_tile - 1) / row_tile;
    const std::uint64_t row_units = checked_mul(checked_mul(num_seqs, p.kv_heads, "4-bit attention batch is too large"),
                                                row_tiles, "4-bit attention batch is too large");
    if (max_count > 1 && (tensor ? rows >= 64 : rows >= 128 && row_units >= 148)) {
        plan.kind = tensor ? Kv4Plan::kTensor : Kv4Plan::kRows;
        plan.columns = static_cast<std::uint32_t>(row_tile);
        plan.column_tiles = static_cast<std::uint32_t>(row_tiles);
        // Up to 1024 CTAs (3.5 waves of two an SM) if all contexts were
        // max_context_len long; the lengths are the device's and most may be
        // shorter, but each split costs a CTA's start and end and a merge. 592,
        // 1024, 2048 and 4096 CTAs: 64 segments of 64 tokens on 1200 263, 263, 379
        // and 380 us, 128 tokens on 120000 739, 715, 799 and 1011, 4 x 512 on zipf
        // 8192 307, 215, 227 and 252.
        const std::uint64_t all = (max_context_len + kv4::kTileTokens - 1) / kv4::kTileTokens;
        std::uint64_t per = p.decode_blocks_per_split;
        if (per == 0) per = std::max<std::uint64_t>(64, checked_mul(row_units, all, "4-bit attention batch is too large") / 1024);
        if (row_units > kMaxSplitUnits) per = all;
        per = (std::max<std::uint64_t>(per, (all + kMaxSplits - 1) / kMaxSplits) + kBlockTiles - 1) / kBlockTiles * kBlockTiles;
        plan.tiles_per_split = static_cast<int>(per);
        plan.max_splits = static_cast<std::uint32_t>((all + per - 1) / per);
        if (row_units > 0x7FFFFFFFull / plan.max_splits) throw std::runtime_error("4-bit attention batch is too large");
        if (plan.max_splits > 1) {
            plan.counter_bytes = kMaxSplitUnits * 4;
            plan.part_bytes = checked_mul(row_units * plan.max_splits, plan.columns * (p.head_dim + 4) * 4, "4-bit attention batch is too large");
        }
        return plan;
    }
    plan.columns = rows <= 4 ? 4 : 8;
    const std::uint64_t column_tiles = (rows + plan.columns - 1) / plan.columns;
    const std::uint64_t units = checked_mul(checked_mul(num_seqs, p.kv_heads, "4-bit attention batch is too large"), column_tiles,
                                            "4-bit attention batch is too large");
    const std::uint32_t tiles = (max_context_len + kv4::kTileTokens - 1) / kv4::kTileTokens;
    std::uint64_t per_split = p.decode_blocks_per_split;
    if (per_split == 0) {
        const std::uint64_t total = checked_mul(units, tiles, "4-bit attention batch is too large");
        if (num_seqs == 1) {
            // Units of one length: two CTAs an SM exactly (131072 tokens x 8
            // kv-heads: 42 us; one or three an SM 60 and 53, four 46).
            per_split = std::max<std::uint64_t>(8, (total + 295) / 296);
        } else {
            // The lengths are the device's: as if all were max_context_len long,
            // two waves of four CTAs an SM (32 x zipf 8192: 103 tiles a split
            // 41 us, 64 and 171 tiles 43 and 52). Where the units alone are two
            // CTAs an SM a split costs more than it evens out below 128 tiles
            // (64 x 64..2048: whole 20.6 us, 64 tiles 23.2), and above 256 one
            // long context would be the tail; segments of many column tiles
            // even that out themselves.
            per_split = std::max<std::uint64_t>(total / 1184, units >= 296 ? 128 : 16);
            per_split = std::min<std::uint64_t>(per_split, 256 * std::max<std::uint64_t>(1, column_tiles / 4));
            // But not more than kMaxSplitCtas, most of which find no keys where
            // the bound is one long context's: 512 sequences x 8 kv-heads of 1000
            // tokens, one of 131072, in 4096 x 8, 16, 32 CTAs 264, 295, 432 us;
            // 2048 of 300 tokens in 16384 x 2, 8, 32 328, 532, 1354 us (one of
            // 131072 among them 611, 562, 1398) and 69 MB, 277 MB, 1.1 GB of
            // partials; 1024 of 500, one of 32768, in 8192 x 2, 4, 8 225, 244, 313.
            const std::uint64_t most = std::max<std::uint64_t>(1, kMaxSplitCtas / units);
            per_split = std::max<std::uint64_t>(per_split, (tiles + most - 1) / most);
        }
        const std::uint64_t splits = (tiles + per_split - 1) / per_split;
        per_split = (tiles + splits - 1) / splits;
    }
    if (units > kMaxSplitUnits) per_split = tiles;
    per_split = std::max<std::uint64_t>(per_split, (tiles + kMaxSplits - 1) / kMaxSplits);
    plan.tiles_per_split = static_cast<int>(per_split);
    plan.max_splits = static_cast<std::uint32_t>((tiles + per_split - 1) / per_split);
    if (units > 0x7FFFFFFFull / plan.max_splits) throw std::runtime_error("4-bit attention batch is too large");
    plan.column_tiles = static_cast<std::uint32_t>(column_tiles);
    if (plan.max_splits > 1) {
        plan.counter_bytes = kMaxSplitUnits * 4;
        plan.part_bytes = checked_mul(units * plan.max_splits, plan.columns * (p.head_dim + 4) * 4, "4-bit attention batch is too large");
    }
    return plan;
}

void check_kv4(const InferlabCudaKvPool& p, const void* queries, std::uint32_t query_dtype,
               std::uint32_t q_heads, std::uint32_t max_blocks, std::uint32_t max_context_len,
               const void* out) {
    if (p.kv_bits != 4) throw std::runtime_error("4-bit attention needs a 4-bit pool");
    if (query_dtype != kFp32 && query_dtype != p.dtype) {
        throw std::runtime_error("4-bit attention query dtype must be FP32 or the pool's row type");
    }
    if (q_heads == 0 || q_heads % p.kv_heads != 0) {
        throw std::runtime_error("4-bit attention q_heads must be a positive multiple of kv_heads");
    }
    if (max_blocks == 0 || max_context_len == 0 || max_context_len > 0x7FFFFF00u) {
        throw std::runtime_error("4-bit attention block table and context bound must be positive");
    }
    if (reinterpret_cast<std::uintptr_t>(queries) % 16 != 0 || reinterpret_cast<std::uintptr_t>(out) % 16 != 0) {
        throw std::runtime_error("4-bit attention queries and output must be 16-byte aligned");
    }
}

void run_kv4(InferlabCudaKvPool& p, Kv4Params k, std::uint32_t query_dtype, std::uint32_t num_seqs,
             std::uint32_t max_context_len, void* workspace, std::size_t workspace_bytes,
             cudaStream_t s) {
    const Kv4Plan plan = plan_kv4(p, num_seqs, k.q_heads, k.max_count, max_context_len, query_dtype);
    if (plan.part_bytes != 0 && (workspace == nullptr || workspace_bytes < plan.counter_bytes + plan.part_bytes)) {
        throw std::runtime_error("4-bit attention workspace is too small");
    }
    if (plan.part_bytes != 0 && reinterpret_cast<std::uintptr_t>(workspace) % 16 != 0) {
        throw std::runtime_error("4-bit attention workspace must be 16-byte aligned");
    }
    k.arena = static_cast<const unsigned char*>(p.key_arena);
    k.num_blocks = p.num_blocks;
    k.kv_heads = p.kv_heads;
    k.group = k.q_heads / p.kv_heads;
    k.tiles_per_block = p.block_tokens / kv4::kTileTokens;
    k.max_context = static_cast<int>(std::min<long long>(max_context_len, static_cast<long long>(k.max_blocks) * p.block_tokens));
    k.column_tiles = plan.column_tiles;
    k.max_splits = plan.max_splits;
    k.per_seq = p.kv_heads * plan.column_tiles;
    // What decides is how much the lengths differ, which only the device knows, and
    // the number of sequences stands in for it. us without / by length, 32 heads
    // over 8 kv-heads x 128, split: a decode of one context of 32768 among short
    // ones 39 / 33 (8 sequences), 57 / 47 (32), 63 / 56 (64); of zipf lengths 106 /
    // 106 (16), 131 / 130 (32), 247 / 250 (64); of 4096 to 32768 evenly drawn 47 /
    // 53 (8), 159 / 174 (32), 270 / 305 (64); of one length 233 / 238 (32). So by
    // length up to 32 costs even batches up to 13% and gives skewed ones up to 18%,
    // and more than 32, which are mostly even, do without. Row tiles (128 tokens
    // each on up to 8192) gain at every size: zipf 826 / 750 (32), 829 / 752 (33),
    // 1610 / 1431 (64), even 960 / 793, 970 / 808, 1714 / 1517, so from 33 on this
    // rule leaves them 10 to 20%. Whole contexts only where the CTAs are not all
    // resident at once (64 x 5 drafted tokens: 78 / 70; row tiles have an order of
    // their own).
    k.by_length = num_seqs > 1 && (plan.max_splits > 1 ? num_seqs <= 32
                                                       : plan.kind == Kv4Plan::kColumns && num_seqs <= 64 &&
                                                             static_cast<std::uint64_t>(num_seqs) * k.per_seq > 592);
    k.tiles_per_split = plan.tiles_per_split;
    k.scale_log2 = kLog2e / std::sqrt(static_cast<float>(p.head_dim));
    k.ws_count = static_cast<std::uint32_t*>(workspace);
    k.ws_part = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + plan.counter_bytes);
    k.error_word = p.error_word;
    k.num_seqs = num_seqs;
    const unsigned grid = num_seqs * k.per_seq * plan.max_splits;
    auto launch = [&](auto row_type, auto query_type) {
        using RowT = decltype(row_type);
        using QT = decltype(query_type);
        const bool wide = p.head_dim == 128;
        void (*kernel)(Kv4Params) = nullptr;
        int smem = kWarps * kRing * kStep * kv4::tile_bytes(static_cast<int>(p.head_dim));
        unsigned threads = kWarps * 32;
        if (plan.kind == Kv4Plan::kColumns) {
            kernel = wide ? (plan.columns == 4 ? kv4_attention_kernel<RowT, QT, 128, true> : kv4_attention_kernel<RowT, QT, 128, false>)
                          : (plan.columns == 4 ? kv4_attention_kernel<RowT, QT, 64, true> : kv4_attention_kernel<RowT, QT, 64, false>);
        } else if constexpr (std::is_same<QT, float>::value) {
            kernel = wide ? kv4_rows_kernel<RowT, 128> : kv4_rows_kernel<RowT, 64>;
            smem = wide ? RowSmem<128>::kBytes : RowSmem<64>::kBytes;
        } else {
            kernel = wide ? kv4_prefill_tc_kernel<QT, 128> : kv4_prefill_tc_kernel<QT, 64>;
            smem = wide ? TcSmem<128>::kBytes : TcSmem<64>::kBytes;
            threads = kTcThreads;
        }
        static std::atomic<std::uint64_t> allowed[2][3];  // devices whose kernel may use it
        auto& devices = allowed[wide][plan.kind != Kv4Plan::kColumns ? 2 : plan.columns == 4];
        const std::uint64_t bit = p.device < 64 ? 1ull << p.device : 0;
        if ((devices.load() & bit) == 0) {
            cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "cudaFuncSetAttribute");
            devices.fetch_or(bit);
        }
        kernel<<<grid, threads, smem, s>>>(k);
    };
    if (p.dtype == kF16) {
        if (query_dtype == kFp32) launch(__half{}, float{});
        else launch(__half{}, __half{});
    } else {
        if (query_dtype == kFp32) launch(__nv_bfloat16{}, float{});
        else launch(__nv_bfloat16{}, __nv_bfloat16{});
    }
    cuda_check(cudaGetLastError(), "4-bit attention launch");
}

}  // namespace
}  // namespace ilb

extern "C" std::size_t inferlab_cuda_kv4_workspace_size(const InferlabCudaKvPool* pool,
                                                        std::uint32_t num_seqs, std::uint32_t q_heads,
                                                        std::uint32_t max_query_count,
                                                        std::uint32_t max_context_len) {
    if (pool == nullptr || pool->kv_bits != 4 || num_seqs == 0 || q_heads < pool->kv_heads ||
        max_query_count == 0 || max_context_len == 0) {
        return 0;
    }
    try {
        // For either type of query.
        std::size_t most = 0;
        for (const std::uint32_t dtype : {ilb::kFp32, ilb::kF16}) {
            const auto plan = ilb::plan_kv4(*pool, num_seqs, q_heads, max_query_count, max_context_len, dtype);
            most = std::max(most, plan.counter_bytes + plan.part_bytes);
        }
        return most;
    } catch (...) {
        return 0;  // the call itself reports why
    }
}

extern "C" int inferlab_cuda_kv4_plan(std::uint32_t kv_heads, std::uint32_t head_dim,
                                      std::uint32_t num_seqs, std::uint32_t q_heads,
                                      std::uint32_t query_dtype, std::uint32_t max_query_count,
                                      std::uint32_t max_context_len, std::uint32_t tiles_per_split,
                                      InferlabCudaKv4Plan* plan, char* error,
                                      std::size_t error_capacity) {
    return ilb::protect(error, error_capacity, [&] {
        if (plan == nullptr) throw std::runtime_error("4-bit attention plan output pointer is null");
        *plan = InferlabCudaKv4Plan{};
        if (kv_heads == 0 || q_heads == 0 || q_heads % kv_heads != 0) {
            throw std::runtime_error("4-bit attention q_heads must be a positive multiple of kv_heads");
        }
        if (head_dim != 64 && head_dim != 128) throw std::runtime_error("4-bit paged KV head_dim must be 64 or 128");
        if (num_seqs == 0 || max_query_count == 0 || max_context_len == 0 || max_context_len > 0x7FFFFF00u) {
            throw std::runtime_error("4-bit attention bounds must be positive");
        }
        if (query_dtype > ilb::kBf16) throw std::runtime_error("4-bit attention query dtype must be FP32 or the pool's row type");
        if (tiles_per_split > 1024) throw std::runtime_error("paged decode split length must be at most 1024 blocks");
        InferlabCudaKvPool shape;
        shape.kv_heads = kv_heads;
        shape.head_dim = head_dim;
        shape.decode_blocks_per_split = tiles_per_split;
        const auto p = ilb::plan_kv4(shape, num_seqs, q_heads, max_query_count, max_context_len, query_dtype);
        plan->kernel = p.kind == ilb::Kv4Plan::kColumns ? 0 : p.kind == ilb::Kv4Plan::kRows ? 1 : 2;
        plan->tile_rows = p.columns;
        plan->max_splits = p.max_splits;
        plan->tokens_per_split = static_cast<std::uint64_t>(p.tiles_per_split) * ilb::kv4::kTileTokens;
        plan->ctas = static_cast<std::uint64_t>(num_seqs) * kv_heads * p.column_tiles * p.max_splits;
        plan->workspace_bytes = p.counter_bytes + p.part_bytes;
    });
}

extern "C" int inferlab_cuda_kv4_decode(InferlabCudaKvPool* pool, const void* queries,
                                        std::uint32_t query_dtype, const std::int32_t* block_tables,
                                        std::uint32_t max_blocks_per_seq,
                                        const std::int32_t* context_lens, std::uint32_t num_seqs,
                                        std::uint32_t q_heads, std::uint32_t max_context_len,
                                        void* out, void* workspace, std::size_t workspace_bytes,
                                        void* stream, char* error, std::size_t error_capacity) {
    return ilb::protect(error, error_capacity, [&] {
        using namespace ilb;
        auto& p = checked_pool(pool);
        if (num_seqs == 0) return;
        if (queries == nullptr || block_tables == nullptr || context_lens == nullptr || out == nullptr) {
            throw std::runtime_error("4-bit attention pointer is null");
        }
        check_kv4(p, queries, query_dtype, q_heads, max_blocks_per_seq, max_context_len, out);
        DeviceGuard guard(p.device);
        Kv4Params k{};
        k.queries = queries;
        k.out = out;
        k.tables = block_tables;
        k.max_blocks = max_blocks_per_seq;
        k.context_lens = context_lens;
        k.max_count = 1;
        k.total_queries = num_seqs;
        k.q_heads = q_heads;
        run_kv4(p, k, query_dtype, num_seqs, max_context_len, workspace, workspace_bytes,
                static_cast<cudaStream_t>(stream));
    });
}

extern "C" int inferlab_cuda_kv4_prefill(InferlabCudaKvPool* pool, const void* queries,
                                         std::uint32_t query_dtype, const std::int32_t* block_tables,
                                         std::uint32_t max_blocks_per_seq,
                                         const std::int32_t* query_starts,
                                         const std::int32_t* query_counts,
                                         const std::int32_t* query_offsets,
                                         std::uint32_t num_segments, std::uint32_t q_heads,
                                         std::uint32_t max_query_count, std::uint64_t total_queries,
                                         std::uint32_t max_context_len, void* out, void* workspace,
                                         std::size_t workspace_bytes, void* stream, char* error,
                                         std::size_t error_capacity) {
    return ilb::protect(error, error_capacity, [&] {
        using namespace ilb;
        auto& p = checked_pool(pool);
        if (num_segments == 0 || total_queries == 0) return;
        if (queries == nullptr || block_tables == nullptr || query_starts == nullptr ||
            query_counts == nullptr || query_offsets == nullptr || out == nullptr) {
            throw std::runtime_error("4-bit attention pointer is null");
        }
        check_kv4(p, queries, query_dtype, q_heads, max_blocks_per_seq, max_context_len, out);
        if (max_query_count == 0) throw std::runtime_error("4-bit attention query bound must be positive");
        if (total_queries > 0x7FFFFFFFull) throw std::runtime_error("4-bit attention batch is too large");
        DeviceGuard guard(p.device);
        Kv4Params k{};
        k.queries = queries;
        k.out = out;
        k.tables = block_tables;
        k.max_blocks = max_blocks_per_seq;
        k.starts = query_starts;
        k.counts = query_counts;
        k.offsets = query_offsets;
        k.max_count = max_query_count;
        k.total_queries = static_cast<long long>(total_queries);
        k.q_heads = q_heads;
        run_kv4(p, k, query_dtype, num_segments, max_context_len, workspace, workspace_bytes,
                static_cast<cudaStream_t>(stream));
    });
}
