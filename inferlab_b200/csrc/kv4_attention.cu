// kv4_attention.cu - attention over a packed 4-bit pool (kv4.cuh): one decode
// step, and several query tokens per sequence.
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
//   output: V codes as bf16, (0x4300 | c) - 136 = c - 8. The weights p scale are
//     split into two bf16 parts (16 bits together, any range).
// The mma computes S^T = K Q^T and O^T = V^T P^T: 16 tokens or dims by 8 query
// columns, so a GQA group of up to 4 fills the columns with its heads' two
// parts, one of 5 to 8 takes two products. P^T's operand layout is S^T's result
// transposed (movmatrix).
//
// What bounds it: HBM, (D + D / 8) bytes a token and kv-head (144 at D = 128,
// 23 bytes a clock and SM), with ~70% of the issue slots behind it. One CTA of
// four warps per (sequence, kv-head, 8 columns, split); every warp streams its
// own 16-token tiles (one bulk copy each) through a ring in shared memory, so
// that the warps never wait for each other before the merge.
#include "common.cuh"
#include "internal.cuh"
#include "kv4.cuh"
#include "pool.cuh"

#include "../../include/inferlab_attention.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace ilb {
namespace {

constexpr int kWarps = 4;
constexpr int kStages = 4;
constexpr float kRescale = 8.0f;       // log2: weights may grow to 2^8 before the maximum moves
constexpr float kNoScore = -3.0e38f;   // running maximum before any key
constexpr std::uint32_t kMaxSplits = 256;

struct Kv4Params {
    const unsigned char* arena;
    std::uint64_t num_blocks;
    std::uint32_t kv_heads, q_heads, group, tiles_per_block;
    const void* queries;
    void* out;
    const std::int32_t* tables;
    std::uint32_t max_blocks;
    long long max_context;
    const std::int32_t* context_lens;  // decode; null: segments
    const std::int32_t* starts;
    const std::int32_t* counts;
    const std::int32_t* offsets;
    std::uint32_t max_count;           // query tokens a sequence may have
    long long total_queries;
    std::uint32_t column_tiles, max_splits;
    int tiles_per_split;
    float scale_log2;
    std::uint32_t* ws_count;  // [unit]
    float* ws_part;           // [unit][split][columns][D + 2]: m, l, o
    std::uint32_t* error_word;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], std::uint32_t a0, std::uint32_t a1,
                                        std::uint32_t a2, std::uint32_t a3, std::uint32_t b0,
                                        std::uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], std::uint32_t a0, std::uint32_t a1,
                                         std::uint32_t a2, std::uint32_t a3, std::uint32_t b0,
                                         std::uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ std::uint32_t transpose8(std::uint32_t x) {
    std::uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ std::uint32_t bf16_pair(float low, float high) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(low, high);
    return *reinterpret_cast<const std::uint32_t*>(&v);
}
// Two codes (bits 0-3 of each half) as bf16 c - 8.
__device__ __forceinline__ std::uint32_t centred_codes(std::uint32_t nibbles) {
    std::uint32_t x = (nibbles & 0x000f000fu) | 0x43004300u;
    __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&x);
    v = __hsub2(v, __float2bfloat162_rn(136.0f));
    return *reinterpret_cast<const std::uint32_t*>(&v);
}
__device__ __forceinline__ std::uint32_t f16_pair(float low, float high) {
    const __half2 v = __floats2half2_rn(low, high);
    return *reinterpret_cast<const std::uint32_t*>(&v);
}
// Token slot (0..7) that sits in row r of an 8-token mma half: r = 2t is token
// t, r = 2t + 1 token 7 - t. Rows 2t of all t (what four lanes read of V at
// once) and rows r of neighbouring r (K) then fall on different banks.
__device__ __forceinline__ int slot_of_row(int r) { return r & 1 ? 7 - (r >> 1) : r >> 1; }

// kHeads4: at most 4 live columns, each twice: columns 4-7 carry the second
// part of the weights of columns 0-3.
template <typename RowT, typename QT, int D, bool kHeads4>
__global__ void __launch_bounds__(kWarps * 32, 4) kv4_attention_kernel(const Kv4Params p) {
    constexpr int kTile = kv4::tile_bytes(D);
    constexpr int kGroups = D / kv4::kGroup;
    constexpr int kWords = D / 32;  // key words of a lane and token
    constexpr int kMt = D / 16;     // 16-dim tiles of the output
    constexpr int kCols = kHeads4 ? 4 : 8;
    constexpr int kRegion = kStages * kTile;  // a warp's ring, and later its state
    static_assert(kCols * (D + 2) * 4 <= kRegion, "a warp's state must fit its ring");
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ std::uint64_t bars[kWarps * kStages];
    __shared__ int failed;
    __shared__ std::uint32_t ticket;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t4 = lane & 3;
    const std::uint32_t split = blockIdx.x % p.max_splits;
    const std::uint32_t unit = blockIdx.x / p.max_splits;
    const std::uint32_t column_tile = unit % p.column_tiles;
    const std::uint32_t kv_head = unit / p.column_tiles % p.kv_heads;
    const std::uint32_t seq = unit / p.column_tiles / p.kv_heads;

    // ---- what this CTA works on: columns r0 .. r0 + live - 1 of the sequence's
    // count * group query rows (token-major), keys 0 .. longest - 1.
    long long start, count, offset;
    bool valid;
    if (p.context_lens != nullptr) {
        const long long ctx = p.context_lens[seq];
        start = ctx - 1;
        count = 1;
        offset = seq;
        valid = ctx >= 0 && ctx <= p.max_context;
        if (!valid && split == 0 && threadIdx.x == 0) flag_error(p.error_word, kErrContext);
    } else {
        start = p.starts[seq];
        count = p.counts[seq];
        offset = p.offsets[seq];
        valid = start >= 0 && count >= 0 && start + count <= p.max_context;
        const bool rows_ok = count >= 0 && count <= p.max_count && offset >= 0 && offset + count <= p.total_queries;
        if (!(valid && rows_ok) && split == 0 && threadIdx.x == 0) flag_error(p.error_word, kErrSegment);
        if (!rows_ok) return;
    }
    const long long r0 = static_cast<long long>(column_tile) * kCols;
    const int live = static_cast<int>(min(static_cast<long long>(kCols), count * p.group - r0));
    if (live <= 0) return;
    auto row_of = [&](int col) {  // the row of queries / out of a live column
        const long long r = r0 + col;
        return (offset + r / p.group) * p.q_heads + kv_head * p.group + r % p.group;
    };
    const long long longest = valid ? start + (r0 + live - 1) / p.group + 1 : 0;
    if (longest == 0) {  // no sequence, or a bad one: zero rows
        if (split == 0) {
            for (int i = threadIdx.x; i < live * D; i += blockDim.x) {
                static_cast<QT*>(p.out)[row_of(i / D) * D + i % D] = Storage<QT>::from_float(0.0f);
            }
        }
        return;
    }
    const int tiles = static_cast<int>((longest + kv4::kTileTokens - 1) / kv4::kTileTokens);
    const int splits = (tiles + p.tiles_per_split - 1) / p.tiles_per_split;
    if (static_cast<int>(split) >= splits) return;
    const int b0 = static_cast<int>(split) * p.tiles_per_split;
    const int nb = min(tiles - b0, p.tiles_per_split);
    const int mine = warp < nb ? (nb - warp + kWarps - 1) / kWarps : 0;  // tiles b0 + warp + 4 i

    // ---- the ring. Lane i holds the arena tile of the warp's tile 32 k + i.
    unsigned char* ring = smem + warp * kRegion;
    std::uint64_t* full = bars + warp * kStages;
    const std::int32_t* table = p.tables + static_cast<std::size_t>(seq) * p.max_blocks;
    auto arena_tile = [&](int i) -> std::uint64_t {
        if (i >= mine) return 0;
        const std::uint32_t tile = static_cast<std::uint32_t>(b0 + warp + kWarps * i);
        std::int32_t block = table[tile / p.tiles_per_block];
        if (block < 0 || static_cast<std::uint64_t>(block) >= p.num_blocks) {
            flag_error(p.error_word, kErrBadBlock);
            block = 0;  // never dereferenced outside the pool
        }
        return (static_cast<std::uint64_t>(block) * p.kv_heads + kv_head) * p.tiles_per_block + tile % p.tiles_per_block;
    };
    std::uint64_t ids = arena_tile(lane), next_ids = 0;
    auto issue = [&](int i, std::uint64_t id) {  // lane 0
        const int stage = i % kStages;
        mbar_arrive_expect_tx(&full[stage], kTile);
        bulk_copy_g2s(ring + stage * kTile, p.arena + id * kTile, kTile, &full[stage]);
    };
    if (lane == 0) {
        for (int s = 0; s < kStages; ++s) mbar_init(&full[s], 1);
        fence_barrier_init();
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
        const std::uint64_t id = __shfl_sync(0xffffffffu, ids, i);
        if (lane == 0 && i < mine) issue(i, id);
    }
    if (threadIdx.x == 0) failed = 0;

    // ---- queries as the B operand: lane holds column g, dims 32 w + 8 t4 + 0..7.
    std::uint32_t qf[kWords][4];
    float q_sum[kGroups][2], factor[2];  // of this lane's result columns 2 t4, 2 t4 + 1
    int limit[2];                        // keys they see
    {
        const int col = kHeads4 ? g & 3 : g;
        float x[kWords][8];
        float most = 0.0f;
        bool bad = false;
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
            if (col < live) {
                const QT* q = static_cast<const QT*>(p.queries) + row_of(col) * D + 32 * w + 8 * t4;
                constexpr int kPer = 16 / sizeof(QT);
#pragma unroll
                for (int c = 0; c < 8 / kPer; ++c) {
                    widen16(reinterpret_cast<const uint4*>(q)[c], &x[w][c * kPer], QT{});
                }
            }
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
            const int cc = kHeads4 ? (2 * t4 + c) & 3 : 2 * t4 + c;
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
    float z[kGroups][2];
    float o[kMt][4];
#pragma unroll
    for (int k = 0; k < kGroups; ++k) z[k][0] = z[k][1] = 0.0f;
#pragma unroll
    for (int i = 0; i < kMt; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    const int slot = slot_of_row(g);
    const std::uint32_t second_part = kHeads4 && t4 >= 2 ? 0xffffffffu : 0u;

    int done = 0;
    for (; done < mine; ++done) {
        if ((done & 31) == 0) {
            if (done > 0) ids = next_ids;
            next_ids = arena_tile(done + 32 + lane);
        }
        const int stage = done % kStages;
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(&full[stage], (done / kStages) & 1, p.error_word))) {
            if (lane == 0) failed = 1;
            break;
        }
        const unsigned char* tile = ring + stage * kTile;
        const int first = (b0 + warp + kWarps * done) * kv4::kTileTokens;

        // S^T: rows are tokens slot, slot + 8; per group of 64 dims.
        float acc[kGroups][4];
#pragma unroll
        for (int k = 0; k < kGroups; ++k) acc[k][0] = acc[k][1] = acc[k][2] = acc[k][3] = 0.0f;
        std::uint32_t k0[kWords], k1[kWords];
        const unsigned char* key = tile + slot * (D / 2) + t4 * (D / 8);
        if constexpr (D == 128) {
            const uint4 a = *reinterpret_cast<const uint4*>(key);
            const uint4 b = *reinterpret_cast<const uint4*>(key + 8 * (D / 2));
            k0[0] = a.x, k0[1] = a.y, k0[2] = a.z, k0[3] = a.w;
            k1[0] = b.x, k1[1] = b.y, k1[2] = b.z, k1[3] = b.w;
        } else {
            const uint2 a = *reinterpret_cast<const uint2*>(key);
            const uint2 b = *reinterpret_cast<const uint2*>(key + 8 * (D / 2));
            k0[0] = a.x, k0[1] = a.y, k1[0] = b.x, k1[1] = b.y;
        }
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
            const std::uint32_t h0 = k0[w] >> 8, h1 = k1[w] >> 8;
            mma_f16(acc[w / 2], k0[w] & 0x000f000fu, k1[w] & 0x000f000fu, h0 & 0x000f000fu, h1 & 0x000f000fu,
                    qf[w][0], qf[w][1]);
            mma_f16(acc[w / 2], k0[w] & 0x00f000f0u, k1[w] & 0x00f000f0u, h0 & 0x00f000f0u, h1 & 0x00f000f0u,
                    qf[w][2], qf[w][3]);
        }
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // (token half, column): log2 scores
        float2 vp[2][kGroups];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int k = 0; k < kGroups; ++k) {
                const float2 kp = kv4::load_pair(tile, kv4::pair_at(D, slot + 8 * h, k, 0));
                vp[h][k] = kv4::load_pair(tile, kv4::pair_at(D, slot + 8 * h, k, 1));
                const float base = fmaf(-8.0f, kp.x, kp.y);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    s[2 * h + c] = fmaf(kp.x, acc[k][2 * h + c], s[2 * h + c]);
                    s[2 * h + c] = fmaf(base, q_sum[k][c], s[2 * h + c]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] *= factor[i & 1];
        if (first + kv4::kTileTokens > shortest) {
            // Slots behind the last key may hold anything; their pairs count as 0.
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int token = first + slot + 8 * h;
#pragma unroll
                for (int c = 0; c < 2; ++c) s[2 * h + c] = token < limit[c] ? s[2 * h + c] : -INFINITY;
                if (token >= longest) {
#pragma unroll
                    for (int k = 0; k < kGroups; ++k) vp[h][k] = make_float2(0.0f, 0.0f);
                }
            }
        }
        const bool grown = fmaxf(s[0], s[2]) > m[0] + kRescale || fmaxf(s[1], s[3]) > m[1] + kRescale;
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float top = fmaxf(s[c], s[2 + c]);
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                top = fmaxf(top, m[c]);
                const float alpha = ex2_ftz(m[c] - top);
                m[c] = top;
                l[c] *= alpha;
#pragma unroll
                for (int k = 0; k < kGroups; ++k) z[k][c] *= alpha;
#pragma unroll
                for (int i = 0; i < kMt; ++i) o[i][c] *= alpha, o[i][2 + c] *= alpha;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[i] = ex2_ftz(s[i] - m[i & 1]);
            l[i & 1] += s[i];
        }

        // P^T as the B operand, per group of dims: weights times scale.
        std::uint32_t pf[kGroups][2][kHeads4 ? 1 : 2];
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float w0 = s[2 * h] * vp[h][k].x, w1 = s[2 * h + 1] * vp[h][k].x;
                z[k][0] = fmaf(s[2 * h], vp[h][k].y, z[k][0]);
                z[k][1] = fmaf(s[2 * h + 1], vp[h][k].y, z[k][1]);
                const std::uint32_t high = bf16_pair(w0, w1);
                if constexpr (kHeads4) {
                    // Columns 4-7: what the first part leaves.
                    const std::uint32_t taken = high & second_part;
                    const float r0_ = w0 - __uint_as_float(taken << 16), r1_ = w1 - __uint_as_float(taken & 0xffff0000u);
                    pf[k][h][0] = transpose8(bf16_pair(r0_, r1_));
                } else {
                    pf[k][h][0] = transpose8(high);
                    pf[k][h][1] = transpose8(bf16_pair(w0 - __uint_as_float(high << 16), w1 - __uint_as_float(high & 0xffff0000u)));
                }
            }
        }
        // O^T += V^T P^T: k index 2 t4 is token t4, 2 t4 + 1 token 7 - t4.
        std::uint32_t v[4][kGroups];
        const int rows[4] = {t4, 7 - t4, 8 + t4, 15 - t4};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned char* at = tile + kv4::value_word(D, rows[i], g);
            if constexpr (D == 128) {
                const uint2 x = *reinterpret_cast<const uint2*>(at);
                v[i][0] = x.x, v[i][1] = x.y;
            } else {
                v[i][0] = *reinterpret_cast<const std::uint32_t*>(at);
            }
        }
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {  // nibbles 0-3, 4-7: dims 8 g + 0..3, + 4..7
                const std::uint32_t a = __byte_perm(v[0][k], v[1][k], half ? 0x7632 : 0x5410);
                const std::uint32_t b = __byte_perm(v[2][k], v[3][k], half ? 0x7632 : 0x5410);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float (&d)[4] = o[4 * k + 2 * half + j];
                    const std::uint32_t a0 = centred_codes(a >> (8 * j)), a1 = centred_codes(a >> (8 * j + 4));
                    const std::uint32_t a2 = centred_codes(b >> (8 * j)), a3 = centred_codes(b >> (8 * j + 4));
                    mma_bf16(d, a0, a1, a2, a3, pf[k][0][0], pf[k][1][0]);
                    if constexpr (!kHeads4) mma_bf16(d, a0, a1, a2, a3, pf[k][0][1], pf[k][1][1]);
                }
            }
        }
        __syncwarp();  // the tile is read
        const std::uint64_t id = __shfl_sync(0xffffffffu, ((done + kStages) & 31) < kStages ? next_ids : ids, (done + kStages) & 31);
        if (lane == 0 && done + kStages < mine) issue(done + kStages, id);
    }
    if (done < mine && lane == 0) {  // a wait ran out: let this warp's own copies land before it leaves
        for (int i = done; i < min(mine, done + kStages); ++i) {
            mbar_wait_bounded(&full[i % kStages], (i / kStages) & 1, p.error_word);
        }
    }
    __syncwarp();

    // ---- a warp's state into its ring: [column][D] output sums, then m and l.
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
            l[c] += __shfl_xor_sync(0xffffffffu, l[c], off);
#pragma unroll
            for (int k = 0; k < kGroups; ++k) z[k][c] += __shfl_xor_sync(0xffffffffu, z[k][c], off);
        }
    }
    float* state = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int i = 0; i < kMt; ++i) {
        if constexpr (kHeads4) {  // both parts of the weights meet
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] += __shfl_xor_sync(0xffffffffu, o[i][e], 2);
        }
        const int dim = 64 * (i / 4) + 8 * g + 2 * (i % 4);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int col = 2 * t4 + c;
            if (col < kCols) {
                *reinterpret_cast<float2*>(state + col * D + dim) =
                    make_float2(o[i][c] + z[i / 4][c], o[i][2 + c] + z[i / 4][c]);
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
    float* part = p.ws_part + (static_cast<std::size_t>(unit) * p.max_splits + split) * kCols * (D + 2);
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
            const bool ok = isfinite(sum) && sum > 0.0f && failed == 0;
            if (!ok) flag_error(p.error_word, kErrNormalizer);
            static_cast<QT*>(p.out)[row_of(col) * D + i % D] = Storage<QT>::from_float(ok ? total / sum : 0.0f);
        } else {
            part[2 * kCols + i] = total;
            if (i % D == 0) part[2 * col] = top, part[2 * col + 1] = sum;
        }
    }
    if (splits == 1) return;

    // ---- the unit's last CTA merges the splits in their order.
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        ticket = atomicAdd(&p.ws_count[unit], 1u);
        if (ticket == static_cast<std::uint32_t>(splits) - 1) p.ws_count[unit] = 0;
    }
    __syncthreads();
    if (ticket != static_cast<std::uint32_t>(splits) - 1) return;
    __threadfence();
    float* weights = reinterpret_cast<float*>(smem);  // [column][split], then 1 / sum per column
    const float* parts = p.ws_part + static_cast<std::size_t>(unit) * p.max_splits * kCols * (D + 2);
    for (int col = warp; col < live; col += kWarps) {
        float top = kNoScore;
        for (int i = lane; i < splits; i += 32) top = fmaxf(top, __ldcg(parts + static_cast<std::size_t>(i) * kCols * (D + 2) + 2 * col));
        top = warp_max(top);
        float sum = 0.0f;
        for (int i = lane; i < splits; i += 32) {
            const float* ml = parts + static_cast<std::size_t>(i) * kCols * (D + 2) + 2 * col;
            const float weight = ex2_ftz(__ldcg(ml) - top);
            weights[col * kMaxSplits + i] = weight;
            sum = fmaf(weight, __ldcg(ml + 1), sum);
        }
        sum = warp_sum(sum);
        const bool ok = isfinite(sum) && sum > 0.0f;
        if (!ok && lane == 0) flag_error(p.error_word, kErrNormalizer);
        if (lane == 0) weights[kCols * kMaxSplits + col] = ok ? 1.0f / sum : 0.0f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < live * D; i += blockDim.x) {
        const int col = i / D;
        float total = 0.0f;
#pragma unroll 8
        for (int k = 0; k < splits; ++k) {
            total = fmaf(weights[col * kMaxSplits + k], __ldcg(parts + static_cast<std::size_t>(k) * kCols * (D + 2) + 2 * kCols + i), total);
        }
        static_cast<QT*>(p.out)[row_of(col) * D + i % D] = Storage<QT>::from_float(total * weights[kCols * kMaxSplits + col]);
    }
}

// Columns a CTA works on, and how the keys are cut.
struct Kv4Plan {
    std::uint32_t columns, column_tiles, max_splits;
    int tiles_per_split;
    std::size_t counter_bytes, part_bytes;
};

Kv4Plan plan_kv4(const InferlabCudaKvPool& p, std::uint32_t num_seqs, std::uint32_t q_heads,
                 std::uint32_t max_count, std::uint32_t max_context_len) {
    Kv4Plan plan{};
    const std::uint64_t rows = static_cast<std::uint64_t>(q_heads / p.kv_heads) * max_count;
    plan.columns = rows <= 4 ? 4 : 8;
    const std::uint64_t column_tiles = (rows + plan.columns - 1) / plan.columns;
    const std::uint64_t units = checked_mul(checked_mul(num_seqs, p.kv_heads, "4-bit attention batch is too large"), column_tiles,
                                            "4-bit attention batch is too large");
    const std::uint32_t tiles = (max_context_len + kv4::kTileTokens - 1) / kv4::kTileTokens;
    // About 2048 CTAs if every context were max_context_len long, each of at
    // least 16 tiles (4 a warp).
    std::uint64_t per_split = p.decode_blocks_per_split;
    if (per_split == 0) {
        const std::uint64_t splits = std::max<std::uint64_t>(1, 2048 / units);
        per_split = std::max<std::uint64_t>(16, (tiles + splits - 1) / splits);
    }
    per_split = std::max<std::uint64_t>(per_split, (tiles + kMaxSplits - 1) / kMaxSplits);
    plan.tiles_per_split = static_cast<int>(per_split);
    plan.max_splits = static_cast<std::uint32_t>((tiles + per_split - 1) / per_split);
    if (units > 0x7FFFFFFFull / plan.max_splits) throw std::runtime_error("4-bit attention batch is too large");
    plan.column_tiles = static_cast<std::uint32_t>(column_tiles);
    if (plan.max_splits > 1) {
        plan.counter_bytes = (units * 4 + 255) & ~std::size_t(255);
        plan.part_bytes = checked_mul(units * plan.max_splits, plan.columns * (p.head_dim + 2) * 4, "4-bit attention batch is too large");
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
    if (max_blocks == 0 || max_context_len == 0 || max_context_len > 0x7FFFFFF0u) {
        throw std::runtime_error("4-bit attention block table and context bound must be positive");
    }
    if (reinterpret_cast<std::uintptr_t>(queries) % 16 != 0 || reinterpret_cast<std::uintptr_t>(out) % 16 != 0) {
        throw std::runtime_error("4-bit attention queries and output must be 16-byte aligned");
    }
}

void run_kv4(InferlabCudaKvPool& p, Kv4Params k, std::uint32_t query_dtype, std::uint32_t num_seqs,
             std::uint32_t max_context_len, void* workspace, std::size_t workspace_bytes,
             cudaStream_t s) {
    const Kv4Plan plan = plan_kv4(p, num_seqs, k.q_heads, k.max_count, max_context_len);
    if (plan.part_bytes != 0 && (workspace == nullptr || workspace_bytes < plan.counter_bytes + plan.part_bytes)) {
        throw std::runtime_error("4-bit attention workspace is too small");
    }
    k.arena = static_cast<const unsigned char*>(p.key_arena);
    k.num_blocks = p.num_blocks;
    k.kv_heads = p.kv_heads;
    k.group = k.q_heads / p.kv_heads;
    k.tiles_per_block = p.block_tokens / kv4::kTileTokens;
    k.max_context = std::min<long long>(max_context_len, static_cast<long long>(k.max_blocks) * p.block_tokens);
    k.column_tiles = plan.column_tiles;
    k.max_splits = plan.max_splits;
    k.tiles_per_split = plan.tiles_per_split;
    k.scale_log2 = kLog2e / std::sqrt(static_cast<float>(p.head_dim));
    k.ws_count = static_cast<std::uint32_t*>(workspace);
    k.ws_part = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + plan.counter_bytes);
    k.error_word = p.error_word;
    const unsigned grid = static_cast<unsigned>(num_seqs * p.kv_heads * plan.column_tiles * plan.max_splits);
    auto launch = [&](auto row_type, auto query_type) {
        using RowT = decltype(row_type);
        using QT = decltype(query_type);
        auto* kernel = p.head_dim == 128
            ? (plan.columns == 4 ? kv4_attention_kernel<RowT, QT, 128, true> : kv4_attention_kernel<RowT, QT, 128, false>)
            : (plan.columns == 4 ? kv4_attention_kernel<RowT, QT, 64, true> : kv4_attention_kernel<RowT, QT, 64, false>);
        const int smem = kWarps * kStages * kv4::tile_bytes(static_cast<int>(p.head_dim));
        cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "cudaFuncSetAttribute");
        kernel<<<grid, kWarps * 32, smem, s>>>(k);
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
        const auto plan = ilb::plan_kv4(*pool, num_seqs, q_heads, max_query_count, max_context_len);
        return plan.counter_bytes + plan.part_bytes;
    } catch (...) {
        return 0;  // the call itself reports why
    }
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
