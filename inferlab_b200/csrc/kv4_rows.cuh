// kv4_rows.cuh - attention of many fp32 query rows per kv-head over a 4-bit pool
// (prompt chunks and prompts): the codes of a 64-token block are widened once
// in shared memory for 64 query rows, instead of once per 8 columns in
// registers (kv4_attention.cu, whose arithmetic this follows, weights in two f16
// parts). 16-bit queries take the tensor cores (kv4_prefill_tc.cuh), whose f16
// keys and values would not do for an fp32 result.
//
// One CTA of four warps takes 64 rows (token-major, the heads of a token
// together) of a (sequence, kv-head), a warp 16 of them. Per block: the four
// packed tiles arrive by cp.async while the block before is worked on; all
// threads widen them to f16 codes, K as c and V as c - 8 in units of 2^-24 and
// 2^-20 (odd pairs of a word; for K the query carries the 2^-4), rows of 2 D
// bytes with 16-byte chunks swizzled by the token; then S = Q K^T and O += P V
// by mma.sync with operands from ldmatrix. A word's eight dims lie in the order
// 0 4 1 5 2 6 3 7, which the contraction of Q and K does not see and O undoes
// when it is stored. The pairs (scale, zero - 8 scale) and (scale, zero) are
// widened to fp32 beside them and applied to scores and weights.
// Bound by shared memory and latency: 16 rows, 16 tokens and 128 dims take 48 mma
// (384 clocks of an SM's quarter), 16 ldmatrix and ~230 other instructions of the
// three warps that a quarter holds; 168 registers, 76 bytes of them spilled at D =
// 128. 64 fresh prompts of 128 tokens, 32 heads over 8 kv-heads: 176 us, 470 in
// column tiles; 4 chunks of 512 tokens on contexts up to 8192 850 us, 8 prompts of
// 1 to 1024 tokens of 16 heads 125 (16-bit queries: 212 and 63).
#pragma once

namespace ilb {
namespace {

constexpr int kRowWarps = 4;
constexpr int kRowTile = 16 * kRowWarps;   // query rows of a CTA
constexpr int kBlockTiles = 4;             // packed tiles of a block
constexpr int kBlockTokens = kBlockTiles * kv4::kTileTokens;

template <int D>
struct RowSmem {
    static constexpr int kRaw = kBlockTiles * kv4::tile_bytes(D);
    static constexpr int kRow = 2 * D;                       // bytes of a token's codes
    static constexpr int kCodes = kBlockTokens * kRow;
    static constexpr int kPairs = kBlockTokens * (D / kv4::kGroup) * 8;
    static constexpr int kKey = 0, kValue = kCodes, kKeyPairs = 2 * kCodes, kValuePairs = kKeyPairs + kPairs;
    static constexpr int kRawAt = kValuePairs + kPairs;
    static constexpr int kBytes = kRawAt + kRaw;
    static_assert(kRowTile * D * 4 <= 2 * kCodes, "the output is staged over the codes");
};

__device__ __forceinline__ void ldmatrix4(std::uint32_t (&r)[4], std::uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(std::uint32_t (&r)[4], std::uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}

template <typename RowT, int D>
__global__ void __launch_bounds__(kRowWarps * 32, 3) kv4_rows_kernel(const Kv4Params p) {
    using L = RowSmem<D>;
    constexpr int kTile = kv4::tile_bytes(D);
    constexpr int kGroups = D / kv4::kGroup;
    constexpr int kUnits = D / 8;  // words of a token's row
    constexpr int kSteps = D / 16;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ std::uint32_t ticket;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;

    // The row tiles with the most keys come first.
    const Work place = work_of<true>(p);
    const std::uint32_t seq = place.seq, split = place.split, work = seq * p.per_seq + place.rest;
    const std::uint32_t row_tile = p.column_tiles - 1 - place.rest / p.kv_heads, kv_head = place.rest % p.kv_heads;
    const bool first_split = split == 0;
    const std::int32_t s_ = p.starts[seq], c_ = p.counts[seq], o_ = p.offsets[seq];
    const std::uint32_t start = static_cast<std::uint32_t>(s_), count = static_cast<std::uint32_t>(c_),
                        offset = static_cast<std::uint32_t>(o_);
    const bool valid = s_ >= 0 && c_ >= 0 && static_cast<long long>(s_) + c_ <= p.max_context;
    const bool rows_ok = c_ >= 0 && count <= p.max_count && o_ >= 0 && static_cast<long long>(o_) + c_ <= p.total_queries;
    if (!(valid && rows_ok) && threadIdx.x == 0 && row_tile == 0 && first_split) flag_error(p.error_word, kErrSegment);
    const std::uint32_t r0 = row_tile * kRowTile;
    if (!rows_ok || r0 >= count * p.group) return;
    const int live = static_cast<int>(min(static_cast<std::uint32_t>(kRowTile), count * p.group - r0));
    auto token_of = [&](int row) { return (r0 + row) / p.group; };
    auto row_of = [&](int row) -> std::size_t {  // the row of queries / out
        const std::uint32_t token = token_of(row);
        return static_cast<std::size_t>(offset + token) * p.q_heads + kv_head * p.group + (r0 + row - token * p.group);
    };
    if (!valid) {
        for (int i = threadIdx.x; first_split && i < live * D; i += blockDim.x) {
            static_cast<float*>(p.out)[row_of(i / D) * D + i % D] = 0.0f;
        }
        return;
    }
    const int longest = static_cast<int>(start + token_of(live - 1) + 1);
    const int tiles = (longest + kv4::kTileTokens - 1) / kv4::kTileTokens;
    const int splits = (tiles + p.tiles_per_split - 1) / p.tiles_per_split;
    if (static_cast<int>(split) >= splits) return;
    const int from = static_cast<int>(split) * (p.tiles_per_split / kBlockTiles);
    const int blocks = min((tiles + kBlockTiles - 1) / kBlockTiles, from + p.tiles_per_split / kBlockTiles);
    const std::int32_t* table = p.tables + static_cast<std::size_t>(seq) * p.max_blocks;
    const std::uint32_t at = smem_u32(smem);

    // Warp w brings tile 4 b + w of block b. Its block id is asked for a block
    // ahead.
    auto id_of = [&](int b) {
        return table[min(static_cast<std::uint32_t>(b * kBlockTiles + warp) / p.tiles_per_block, p.max_blocks - 1)];
    };
    auto fetch = [&](int b, std::int32_t block) {
        const int tile = b * kBlockTiles + warp;
        if (tile < tiles) {
            if (block < 0 || static_cast<std::uint64_t>(block) >= p.num_blocks) {
                if (lane == 0) flag_error(p.error_word, kErrBadBlock);
                block = 0;  // never dereferenced outside the pool
            }
            const std::uint64_t index = (static_cast<std::uint64_t>(block) * p.kv_heads + kv_head) * p.tiles_per_block +
                                        static_cast<std::uint32_t>(tile) % p.tiles_per_block;
            const unsigned char* src = p.arena + index * kTile + lane * 16;
            const std::uint32_t to = at + L::kRawAt + warp * kTile + lane * 16;
#pragma unroll
            for (int c = 0; c < kTile; c += 512) {
                if (c + 512 <= kTile || lane * 16 < kTile - c) cp_async16(to + c, src + c);
            }
        }
        cp_async_commit();
    };
    std::int32_t next_id = id_of(from);
    fetch(from, next_id);
    next_id = id_of(from + 1);

    // ---- queries, as in kv4_attention.cu: rows g and g + 8 of the warp's 16,
    // scaled by a power of two, f16 in the codes' order and units, staged where
    // the keys go.
    float q_sum[2][kGroups], factor[2];
    int limit[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = 16 * warp + 8 * h + g;
        const float* src = static_cast<const float*>(p.queries) + row_of(min(row, live - 1)) * D + 8 * t4;
        float x[D / 32][8], most = 0.0f;
        bool bad = false;
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
#pragma unroll
            for (int c = 0; c < 2; ++c) widen16(reinterpret_cast<const uint4*>(src + 32 * w)[c], &x[w][4 * c], 0.0f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[w][i] = row < live ? Storage<RowT>::to_float(Storage<RowT>::from_float(x[w][i])) : 0.0f;
                bad |= !isfinite(x[w][i]);
                most = fmaxf(most, fabsf(x[w][i]));
            }
        }
        if (bad) flag_error(p.error_word, kErrNonFinite);
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int exponent = max(15, static_cast<int>(__float_as_uint(most) >> 23));
        const float up = most > 0.0f ? __uint_as_float(static_cast<std::uint32_t>(min(254, 268 - exponent)) << 23) : 1.0f;
        factor[h] = fminf(p.scale_log2 * 16777216.0f / up, 3.0e38f);
        limit[h] = row < live ? static_cast<int>(start + token_of(row) + 1) : 0;
#pragma unroll
        for (int k = 0; k < kGroups; ++k) q_sum[h][k] = 0.0f;
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[w][i] *= up;
                q_sum[h][w / 2] += x[w][i];
            }
            const uint4 word = make_uint4(f16_pair(x[w][0], x[w][4]), f16_pair(x[w][1] * 0.0625f, x[w][5] * 0.0625f),
                                          f16_pair(x[w][2], x[w][6]), f16_pair(x[w][3] * 0.0625f, x[w][7] * 0.0625f));
            const int unit = 4 * w + t4;
            *reinterpret_cast<uint4*>(smem + L::kKey + row * L::kRow + ((unit ^ (row & 7)) << 4)) = word;
        }
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
            q_sum[h][k] += __shfl_xor_sync(0xffffffffu, q_sum[h][k], 1);
            q_sum[h][k] += __shfl_xor_sync(0xffffffffu, q_sum[h][k], 2);
            q_sum[h][k] *= 5.9604644775390625e-08f;  // 2^-24
        }
    }
    __syncwarp();
    std::uint32_t qf[kSteps][4];
    {
        const int row = 16 * warp + (lane & 15);  // matrices: rows 0-7, 8-15 of word 2 s, then of word 2 s + 1
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int unit = 2 * s + (lane >> 4);
            ldmatrix4(qf[s], at + L::kKey + row * L::kRow + ((unit ^ (row & 7)) << 4));
        }
    }
    // Keys that all, and that any, of the warp's rows see.
    const int first_row = 16 * warp, last_row = min(16 * warp + 15, live - 1);
    const int clear = first_row < live ? static_cast<int>(start + token_of(first_row) + 1) : 0;
    const int reach = first_row < live ? static_cast<int>(start + token_of(last_row) + 1) : 0;

    float m[2] = {kNoScore, kNoScore};
    float2 l2[2], z2[2][kGroups];  // sums of even and odd tokens
    float o[kUnits][4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l2[r] = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < kGroups; ++k) z2[r][k] = make_float2(0.0f, 0.0f);
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    // ldmatrix rows of this lane: keys (tokens 0-7 of words 2 s, 2 s + 1, then
    // tokens 8-15), values (tokens 0-15 of word u, then of word u + 1).
    const int key_token = (lane & 7) + ((lane >> 4) << 3), key_unit = (lane >> 3) & 1;
    const int value_token = lane & 15, value_unit = lane >> 4;

    for (int b = from; b < blocks; ++b) {
        cp_async_wait_group<0>();
        __syncthreads();  // the block is here, and the codes before it are used
        // ---- widen: 16 bytes (four words) of a code row at a time.
#pragma unroll
        for (int i = 0; i < kBlockTokens * kUnits / 4 / (kRowWarps * 32); ++i) {
            const int n = threadIdx.x + i * kRowWarps * 32;
            const int token = n / (kUnits / 4), part = n % (kUnits / 4);
            const unsigned char* tile = smem + L::kRawAt + token / kv4::kTileTokens * kTile;
            const int slot = token % kv4::kTileTokens;
            const uint4 key = *reinterpret_cast<const uint4*>(tile + slot * (D / 2) + part * 16);
            const uint4 value = *reinterpret_cast<const uint4*>(tile + kv4::half_tile_bytes(D) + slot * (D / 2) + part * 16);
            const std::uint32_t kw[4] = {key.x, key.y, key.z, key.w}, vw[4] = {value.x, value.y, value.z, value.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // Word 4 part + j of the row: its dims' unit, from kv4.cuh's order.
                const int w = 4 * part + j;
                const int ku = ((w % (D / 32)) << 2) + w / (D / 32);
                const int chunk = w / kGroups ^ (D == 128 ? ((slot >> 1) & 1) * 4 : 0);
                const int vu = (w % kGroups) * 8 + chunk;
                const std::uint32_t kh = kw[j] >> 8, vh = vw[j] >> 8;
                *reinterpret_cast<uint4*>(smem + L::kKey + token * L::kRow + ((ku ^ (token & 7)) << 4)) =
                    make_uint4(kw[j] & 0x000f000fu, kw[j] & 0x00f000f0u, kh & 0x000f000fu, kh & 0x00f000f0u);
                *reinterpret_cast<uint4*>(smem + L::kValue + token * L::kRow + ((vu ^ (token & 7)) << 4)) =
                    make_uint4(centred_low(vw[j]), centred_high(vw[j]), centred_low(vh), centred_high(vh));
            }
        }
        for (int n = threadIdx.x; n < 2 * kBlockTokens * kGroups; n += kRowWarps * 32) {
            const int which = n / (kBlockTokens * kGroups), i = n % (kBlockTokens * kGroups);
            const int token = i / kGroups, k = i % kGroups;
            float2 pair = kv4::load_pair(smem + L::kRawAt + token / kv4::kTileTokens * kTile,
                                         kv4::pair_at(D, token % kv4::kTileTokens, k, which));
            if (which == 0) pair.y = fmaf(-8.0f, pair.x, pair.y);
            // Slots behind the last key may hold anything.
            if (b * kBlockTokens + token >= longest) pair = make_float2(0.0f, 0.0f);
            float* to = reinterpret_cast<float*>(smem + (which ? L::kValuePairs : L::kKeyPairs)) +
                        ((token >> 1) * kGroups + k) * 4 + (token & 1);
            to[0] = pair.x, to[2] = pair.y;
        }
        __syncthreads();
        if (b + 1 < blocks) {
            fetch(b + 1, next_id);
            next_id = id_of(b + 2);
        }

#pragma unroll 1
        for (int t0 = 0; t0 < kBlockTokens; t0 += 16) {
            const int first = b * kBlockTokens + t0;
            if (first >= reach) break;
            // S: rows g, g + 8; tokens 2 t4, 2 t4 + 1 of two halves; per group.
            float acc[kGroups][2][4];
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                std::uint32_t kf[4];
                const int token = t0 + key_token, unit = 2 * s + key_unit;
                ldmatrix4(kf, at + L::kKey + token * L::kRow + ((unit ^ (token & 7)) << 4));
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float (&d)[4] = acc[s / 4][h];
                    if (s % 4 == 0) mma_f16_first(d, qf[s][0], qf[s][1], qf[s][2], qf[s][3], kf[2 * h], kf[2 * h + 1]);
                    else mma_f16(d, qf[s][0], qf[s][1], qf[s][2], qf[s][3], kf[2 * h], kf[2 * h + 1]);
                }
            }
            // Two tokens an instruction from here on.
            float2 s[2][2], vs[2][kGroups], vz[2][kGroups];  // log2 scores by half and row; value pairs
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at_pair = (t0 / 2 + 4 * h + t4) * kGroups * 16;
#pragma unroll
                for (int k = 0; k < kGroups; ++k) {
                    const float4 key = *reinterpret_cast<const float4*>(smem + L::kKeyPairs + at_pair + 16 * k);
                    const float4 value = *reinterpret_cast<const float4*>(smem + L::kValuePairs + at_pair + 16 * k);
                    vs[h][k] = make_float2(value.x, value.y), vz[h][k] = make_float2(value.z, value.w);
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float2 sum = make_float2(q_sum[r][k], q_sum[r][k]);
                        s[h][r] = k == 0 ? kv4::mul2(make_float2(key.z, key.w), sum) : kv4::fma2(make_float2(key.z, key.w), sum, s[h][r]);
                        s[h][r] = kv4::fma2(make_float2(key.x, key.y), make_float2(acc[k][h][2 * r], acc[k][h][2 * r + 1]), s[h][r]);
                    }
                }
#pragma unroll
                for (int r = 0; r < 2; ++r) s[h][r] = kv4::mul2(s[h][r], make_float2(factor[r], factor[r]));
            }
            if (first + 16 > clear) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int token = first + 8 * h + 2 * t4;
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        if (token >= limit[r]) s[h][r].x = -INFINITY;
                        if (token + 1 >= limit[r]) s[h][r].y = -INFINITY;
                    }
                }
            }
            // Weights against m and times the value scales, as in kv4_attention.cu.
            float2 weight[2][2], scaled[2][kGroups][2];
            float most_weight = 0.0f, most_scaled = 0.0f;
            auto weigh = [&] {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        // Subtracted from the rounded score: m is one of those less the
                        // headroom, and large scores differ from theirs by more.
                        weight[h][r] = make_float2(ex2_ftz(__fsub_rn(s[h][r].x, m[r])), ex2_ftz(__fsub_rn(s[h][r].y, m[r])));
                        most_weight = fmax3(most_weight, weight[h][r].x, weight[h][r].y);
#pragma unroll
                        for (int k = 0; k < kGroups; ++k) {
                            scaled[h][k][r] = kv4::mul2(weight[h][r], vs[h][k]);
                            most_scaled = fmax3(most_scaled, scaled[h][k][r].x, scaled[h][k][r].y);
                        }
                    }
                }
            };
            weigh();
            if (__any_sync(0xffffffffu, most_scaled > 32768.0f || most_weight > 17179869184.0f)) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float top = kNoScore;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float2 scale = make_float2(9.5367431640625e-07f, 9.5367431640625e-07f);  // 2^-20
#pragma unroll
                        for (int k = 0; k < kGroups; ++k) {
                            scale = make_float2(fmaxf(scale.x, vs[h][k].x), fmaxf(scale.y, vs[h][k].y));
                        }
                        top = fmaxf(top, score_with_room(s[h][r].x, __log2f(scale.x)));
                        top = fmaxf(top, score_with_room(s[h][r].y, __log2f(scale.y)));
                    }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    top = fmaxf(top, m[r]);
                    const float alpha = ex2_ftz(m[r] - top);
                    m[r] = top;
                    const float2 both = make_float2(alpha, alpha);
                    l2[r] = kv4::mul2(l2[r], both);
#pragma unroll
                    for (int k = 0; k < kGroups; ++k) z2[r][k] = kv4::mul2(z2[r][k], both);
#pragma unroll
                    for (int i = 0; i < kUnits; ++i) o[i][2 * r] *= alpha, o[i][2 * r + 1] *= alpha;
                }
                weigh();
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    l2[r] = kv4::add2(l2[r], weight[h][r]);
#pragma unroll
                    for (int k = 0; k < kGroups; ++k) z2[r][k] = kv4::fma2(weight[h][r], vz[h][k], z2[r][k]);
                }
            }
            // O += P V: A = P (rows g, g + 8; tokens of the halves).
#pragma unroll
            for (int k = 0; k < kGroups; ++k) {
                std::uint32_t a[4], a2[4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float w0 = scaled[h][k][r].x, w1 = scaled[h][k][r].y;
                        a[2 * h + r] = f16_pair(w0, w1);
                        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&a[2 * h + r]));
                        a2[2 * h + r] = f16_pair(w0 - t.x, w1 - t.y);
                    }
                }
#pragma unroll
                for (int u = 8 * k; u < 8 * k + 8; u += 2) {
                    std::uint32_t vf[4];
                    const int token = t0 + value_token, unit = u + value_unit;
                    ldmatrix4_trans(vf, at + L::kValue + token * L::kRow + ((unit ^ (token & 7)) << 4));
                    mma_f16(o[u], a[0], a[1], a[2], a[3], vf[0], vf[1]);
                    mma_f16(o[u + 1], a[0], a[1], a[2], a[3], vf[2], vf[3]);
                    mma_f16(o[u], a2[0], a2[1], a2[2], a2[3], vf[0], vf[1]);
                    mma_f16(o[u + 1], a2[0], a2[1], a2[2], a2[3], vf[2], vf[3]);
                }
            }
        }
    }

    // ---- output rows, staged over the codes in dim order; a split's sums go to
    // the workspace instead, and the last of a row tile's CTAs merges them.
    __syncthreads();
    float l[2], z[2][kGroups], inv[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] = l2[r].x + l2[r].y;
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
            z[r][k] = z2[r][k].x + z2[r][k].y;
            z[r][k] += __shfl_xor_sync(0xffffffffu, z[r][k], 1);
            z[r][k] += __shfl_xor_sync(0xffffffffu, z[r][k], 2);
        }
        const bool ok = isfinite(l[r]) && l[r] > 0.0f;
        if (splits == 1 && !ok && 16 * warp + 8 * r + g < live) flag_error(p.error_word, kErrNormalizer);
        inv[r] = splits > 1 ? 1.0f : ok ? 1.0f / l[r] : 0.0f;
    }
    const float unit = t4 % 2 ? 1048576.0f : 16777216.0f;  // back from the codes' 2^-20, 2^-24
    float* stage = reinterpret_cast<float*>(smem) + 16 * warp * D;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                stage[(8 * r + g) * D + 8 * u + t4 + 4 * c] = fmaf(o[u][2 * r + c], unit, z[r][u / 8]) * inv[r];
            }
        }
    }
    __syncwarp();
    constexpr int kPart = kRowTile * (D + 4);
    float* part = p.ws_part + (static_cast<std::size_t>(work) * p.max_splits + split) * kPart;
    if (splits > 1 && t4 == 0) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            *reinterpret_cast<float2*>(part + kRowTile * D + 2 * (16 * warp + 8 * r + g)) = make_float2(m[r], l[r]);
        }
    }
    for (int i = lane; i < 16 * D / 4; i += 32) {
        const int row = 16 * warp + i / (D / 4);
        if (row >= live) break;
        const float4 x = *reinterpret_cast<const float4*>(stage + 4 * i);
        if (splits > 1) {
            *reinterpret_cast<float4*>(part + 16 * warp * D + 4 * i) = x;
            continue;
        }
        store_row4(static_cast<float*>(p.out) + row_of(row) * D + 4 * i % D, x);
    }
    if (splits == 1) return;
    if (!last_of(p.ws_count + work, splits, ticket)) return;
    const float* parts = p.ws_part + static_cast<std::size_t>(work) * p.max_splits * kPart;
    for (int i = threadIdx.x; i < live * D / 4; i += blockDim.x) {
        const int row = i / (D / 4);
        bool ok;
        const float4 x = merge_parts<kPart, kRowTile * D>(parts, splits, row, i, ok);
        if (!ok) flag_error(p.error_word, kErrNormalizer);
        store_row4(static_cast<float*>(p.out) + row_of(row) * D + 4 * i % D, x);
    }
}

}  // namespace
}  // namespace ilb
