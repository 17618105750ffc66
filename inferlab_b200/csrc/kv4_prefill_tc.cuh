// kv4_prefill_tc.cuh - attention of many 16-bit query rows per kv-head over a
// 4-bit pool on the sm_100a tensor cores.
//
// One CTA of 256 threads takes 128 rows (token-major, the heads of a token
// together) of a (sequence, kv-head) and a split of its keys, 64 keys a block.
// Two threads own a row, one for each half of a block's keys:
//   scores   S = Q K^T from TMEM into registers, the row's largest;
//   weights  p against m and p 2^e as f16 back over S, where the next MMA reads
//     them. O stays in TMEM and is rescaled only when a row's largest p 2^e
//     leaves f16's upper range;
//   widen    while O += P V of this block and S of the next run, K of the block
//     after that and V of the next: zero + (c - 8) scale as f16 in units of 2^e,
//     a power of two per token that brings the token's largest value below 2^15,
//     64 dims to a 128-byte row with the swizzle that the MMA descriptors name. A
//     word's eight dims lie in the order 0 4 1 5 2 6 3 7, which the contraction of
//     Q and K does not see and O undoes when it is stored. The packed tiles
//     come by cp.async during the weights.
// Rounded to f16 (2^-11): keys, values and p 2^e. For a 16-bit result that is
// the step, or an eighth of it, in which a 16-bit pool would have kept the keys
// and values. Codes with the pairs applied to fp32 scores and weights, as in
// kv4_attention.cu, would be exact, but a thread that owns a row then reads eight
// numbers a key from shared memory instead of two: 426 us for 4 chunks of 512
// tokens on contexts up to 8192.
// Two CTAs an SM: one's softmax runs beside the other's MMAs (half of the 512
// TMEM columns and 110 KB of shared memory each).
// Bound by latency: 54% of the issue slots, 18% of the tensor pipe and 2% of DRAM
// are used. A block is one chain (S, softmax, weights to TMEM, O) with two or three
// barriers of the CTA; it costs the eight warps ~700 instructions each, 250 of them
// the widening, and 4300 clocks, of which only the other CTA uses the gaps. 4
// chunks of 512 tokens on contexts up to 8192, 32 heads over 8 kv-heads: 212 us,
// 376 TFLOP/s. A CTA's queries, first keys and outputs cost as much as four
// blocks, so short prompts come off worse (8 of 1 to 1024 tokens, 16 heads: 63
// us). A second S in TMEM, issued a block ahead, changed nothing.
#pragma once

#include "tc_common.cuh"

namespace ilb {
namespace {

constexpr int kTcRows = 128;     // query rows of a CTA
constexpr int kTcKeys = kBlockTokens;
constexpr int kTcThreads = 256;

template <int D>
struct TcSmem {
    static constexpr int kGroups = D / kv4::kGroup;
    static constexpr int kQGroup = kTcRows * 128, kKeyGroup = kTcKeys * 128;  // 64 dims of all rows
    static constexpr int kStage = kGroups * kKeyGroup;
    static constexpr int kScaleBytes = kTcKeys * 4;  // 2^e of every token
    static constexpr int kQ = 0, kK = kGroups * kQGroup, kV = kK + 2 * kStage, kKeyScales = kV + 2 * kStage;
    static constexpr int kValueScales = kKeyScales + 2 * kScaleBytes;
    static constexpr int kTops = kValueScales + 2 * kScaleBytes, kRaw = kTops + 2 * kTcRows * 4;
    static constexpr int kBars = kRaw + kBlockTiles * kv4::tile_bytes(D);
    static constexpr int kBytes = kBars + 16 + 1024;  // aligned by hand
    static_assert(kBlockTiles * kv4::half_tile_bytes(D) <= kStage, "the first raw keys lie in a stage");
    static_assert(kTcRows * D * 4 <= kV - kQ && 2 * kTcRows * 4 <= kStage, "the output lies over queries and keys");
    static constexpr int kTmem = D == 128 ? 256 : 128;  // columns: S, then O (a power of two)
};
enum { kTcS = 0, kTcDone, kTcBars };

__device__ __forceinline__ void tmem_load16(std::uint32_t at, std::uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at));
}
// Names the registers, so that no use of them comes before the load.
__device__ __forceinline__ void tmem_wait16(std::uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// One lane of a converged warp, the same for all of its lanes.
__device__ __forceinline__ bool elect_one() {
    std::uint32_t chosen;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(chosen));
    return chosen != 0;
}

template <typename QT, int D>
__global__ void __launch_bounds__(kTcThreads, 2) kv4_prefill_tc_kernel(const Kv4Params p) {
    using L = TcSmem<D>;
    constexpr int kTile = kv4::tile_bytes(D);
    constexpr int kGroups = L::kGroups;
    constexpr int kUnits = D / 8;  // words of a token's row
    extern __shared__ unsigned char tc_smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<std::uintptr_t>(tc_smem_raw) + 1023) &
                                                           ~static_cast<std::uintptr_t>(1023));
    auto* bars = reinterpret_cast<std::uint64_t*>(smem + L::kBars);
    __shared__ std::uint32_t ticket, tmem_at;
    __shared__ int abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

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
    const std::uint32_t r0 = row_tile * kTcRows;
    if (!rows_ok || r0 >= count * p.group) return;
    const int live = static_cast<int>(min(static_cast<std::uint32_t>(kTcRows), count * p.group - r0));
    auto token_of = [&](int row) { return (r0 + row) / p.group; };
    auto row_of = [&](int row) -> std::size_t {  // the row of queries / out
        const std::uint32_t token = token_of(row);
        return static_cast<std::size_t>(offset + token) * p.q_heads + kv_head * p.group + (r0 + row - token * p.group);
    };
    if (!valid) {
        for (int i = threadIdx.x; first_split && i < live * D; i += blockDim.x) {
            static_cast<QT*>(p.out)[row_of(i / D) * D + i % D] = Storage<QT>::from_float(0.0f);
        }
        return;
    }
    const int longest = static_cast<int>(start + token_of(live - 1) + 1);
    const int tiles = (longest + kv4::kTileTokens - 1) / kv4::kTileTokens;
    const int splits = (tiles + p.tiles_per_split - 1) / p.tiles_per_split;
    if (static_cast<int>(split) >= splits) return;
    const int from = static_cast<int>(split) * (p.tiles_per_split / kBlockTiles);
    const int blocks = min((tiles + kBlockTiles - 1) / kBlockTiles, from + p.tiles_per_split / kBlockTiles) - from;
    const std::uint32_t at = smem_u32(smem);

    if (threadIdx.x == 0) {
        mbar_init(&bars[kTcS], 1 + kTcThreads / 32);  // S (and O before it), and every warp's widening
        mbar_init(&bars[kTcDone], 1);
        abort = 0;
        fence_barrier_init();
    }
    if (warp == 0) {
        tc::tmem_alloc(&tmem_at, L::kTmem);
        tc::tmem_relinquish();
    }
    // A thread's row, and where it is in queries and out. A warp's 16 rows of a
    // copy are its own half of the 32 it owns, so that their places are known
    // without a division each.
    const int row = threadIdx.x % kTcRows, half = threadIdx.x / kTcRows;
    const std::uint32_t row_at = static_cast<std::uint32_t>(row_of(min(row, live - 1)) - static_cast<std::size_t>(offset) * p.q_heads);
    auto copied_row = [&](int i, int lanes) { return 16 * half + i * (32 / lanes) + lane / lanes; };  // within the warp's 32
    auto place_of = [&](int r) { return static_cast<std::size_t>(offset) * p.q_heads + __shfl_sync(0xffffffffu, row_at, r); };
    // The queries come as they are to where they go; 16-byte chunks of 64 dims of
    // a row, swizzled.
    auto query_at = [&](int r, int unit) { return L::kQ + (unit / 8) * L::kQGroup + r * 128 + ((unit % 8 ^ (r & 7)) << 4); };
#pragma unroll
    for (int i = 0; i < kUnits / 2; ++i) {
        const int r = copied_row(i, kUnits), unit = lane % kUnits;
        cp_async16(at + query_at(32 * (warp & 3) + r, unit), static_cast<const QT*>(p.queries) + place_of(r) * D + unit * 8);
    }
    cp_async_commit();
    // Warp w brings the keys of tile w of a block, warp 4 + w the values of the
    // block before, block after block; the next one's id is asked for a block
    // ahead. Tiles within a pool block are counted, not divided for.
    const std::int32_t* table = p.tables + static_cast<std::size_t>(seq) * p.max_blocks;
    std::uint32_t tile = static_cast<std::uint32_t>(from * kBlockTiles + (warp & 3));
    std::uint32_t in_block = tile % p.tiles_per_block, pool_block = tile / p.tiles_per_block;
    const std::uint32_t block_step = kBlockTiles / p.tiles_per_block, tile_step = kBlockTiles % p.tiles_per_block;
    const std::uint32_t stop = min(static_cast<std::uint32_t>(tiles), static_cast<std::uint32_t>((from + blocks) * kBlockTiles));
    std::int32_t next_id = table[min(pool_block, p.max_blocks - 1)];
    auto fetch = [&](std::uint32_t raw) {
        if (tile < stop) {
            std::int32_t block = next_id;
            if (block < 0 || static_cast<std::uint64_t>(block) >= p.num_blocks) {
                if (lane == 0) flag_error(p.error_word, kErrBadBlock);
                block = 0;  // never dereferenced outside the pool
            }
            const std::uint64_t index = (static_cast<std::uint64_t>(block) * p.kv_heads + kv_head) * p.tiles_per_block + in_block;
            constexpr int kHalf = kv4::half_tile_bytes(D);
            const unsigned char* src = p.arena + index * kTile + (warp < 4 ? 0 : kHalf) + lane * 16;
            const std::uint32_t to = raw + warp * kHalf + lane * 16;
#pragma unroll
            for (int c = 0; c < kHalf; c += 512) {
                if (c + 512 <= kHalf || lane * 16 < kHalf - c) cp_async16(to + c, src + c);
            }
        }
        tile += kBlockTiles;
        in_block += tile_step;
        pool_block += block_step;
        if (in_block >= p.tiles_per_block) in_block -= p.tiles_per_block, ++pool_block;
        next_id = table[min(pool_block, p.max_blocks - 1)];
    };
    // The first keys come into a stage that is not used yet, so that two blocks
    // are on their way at once.
    constexpr int kFirst = L::kV + L::kStage;
    if (warp < 4) fetch(at + kFirst);
    cp_async_commit();
    fetch(at + L::kRaw);
    cp_async_commit();

    // Widens a code row's 16 bytes (four words) of keys or values.
    constexpr int kItems = kTcKeys * kUnits / 4;
    const int item = threadIdx.x % kItems, index = item / (kUnits / 4), part16 = item % (kUnits / 4);
    // Eight lanes that store at once hold rows whose numbers differ by an odd
    // number across 4, so that their swizzled chunks differ.
    const int token = (index & ~7) + ((index & 7) >> 1 ^ (index & 1) * 5), slot = token % kv4::kTileTokens;
    // Word 4 part16 + j holds the dims of unit (base ^ bits(j)) % 8 of group(j)
    // (kv4.cuh's order): where that is in a swizzled row.
    const int key_at = token * 128 + (((part16 << (D == 128 ? 0 : 1)) ^ (token & 7)) << 4);
    const int value_at = token * 128 + (((part16 << (D == 128 ? 1 : 2)) ^ (D == 128 ? (slot & 2) << 1 : 0) ^ (token & 7)) << 4);
    auto widen_row = [&](const unsigned char* tile, unsigned char* to, float* scales, bool seen, auto values_too) {
        constexpr bool kValue = decltype(values_too)::value;
        const uint4 x = *reinterpret_cast<const uint4*>(tile + slot * (D / 2) + part16 * 16);
        const std::uint32_t word[4] = {x.x, x.y, x.z, x.w};
        float2 pair[kGroups];
        float most = 0.0f;
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
            pair[k] = kv4::load_pair(tile, kv4::pair_at(D, slot, k, 0));
            if (!seen) pair[k] = make_float2(0.0f, 0.0f);  // slots behind the last key may hold anything
            most = fmax3(most, fabsf(fmaf(-8.0f, pair[k].x, pair[k].y)), fabsf(fmaf(7.0f, pair[k].x, pair[k].y)));
        }
        // 2^e: the largest value becomes 2^14 to 2^15, one below 2^-10 less (the
        // f16 pairs are multiples of 2^-24, so nothing is lost): where large
        // scores leave m no room a weight is kept as 2^e, which f16 must hold.
        const std::uint32_t exponent = max(117u, __float_as_uint(most) >> 23);
        const float down = __uint_as_float((268u - exponent) << 23);
        __half2 scale[kGroups], zero[kGroups];
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
            scale[k] = __float2half2_rn(pair[k].x * down);
            zero[k] = __float2half2_rn(pair[k].y * down);
        }
        // 1024 + c and 1024 + 16 c by their bits, so c - 8 exactly.
        const __half2 low_off = __float2half2_rn(-1032.0f), high_unit = __float2half2_rn(0.0625f), high_off = __float2half2_rn(-72.0f);
        auto values = [&](std::uint32_t bits, bool high, int k) {
            bits = (bits & (high ? 0x00f000f0u : 0x000f000fu)) | 0x64006400u;
            const __half2 h = *reinterpret_cast<const __half2*>(&bits);
            const __half2 v = __hfma2(high ? __hfma2(h, high_unit, high_off) : __hadd2(h, low_off), scale[k], zero[k]);
            return *reinterpret_cast<const std::uint32_t*>(&v);
        };
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int bits = kValue ? (D == 128 ? j >> 1 : j) : (j & 1) << 2 | (D == 128 ? 0 : j >> 1);
            const int k = D == 128 ? (kValue ? j & 1 : j >> 1) : 0;
            const std::uint32_t high = word[j] >> 8;
            *reinterpret_cast<uint4*>(to + k * L::kKeyGroup + ((kValue ? value_at : key_at) ^ bits << 4)) =
                make_uint4(values(word[j], false, k), values(word[j], true, k), values(high, false, k), values(high, true, k));
        }
        if (part16 == 0) scales[token] = __uint_as_float((exponent - 14u) << 23);
    };
    // The raw keys become block `key_block`, the raw values the one before.
    auto widen = [&](int key_block, int raw) {
        const int value_block = key_block - 1;
        const unsigned char* tile = smem + raw + token / kv4::kTileTokens * kv4::half_tile_bytes(D);
        if (key_block < blocks && (kItems == kTcThreads || threadIdx.x < kItems)) {
            widen_row(tile, smem + L::kK + (key_block & 1) * L::kStage,
                      reinterpret_cast<float*>(smem + L::kKeyScales + (key_block & 1) * L::kScaleBytes),
                      (from + key_block) * kTcKeys + token < longest,
                      std::false_type{});
        }
        if (value_block >= 0 && value_block < blocks && (kItems == kTcThreads || threadIdx.x >= kItems)) {
            widen_row(tile + kBlockTiles * kv4::half_tile_bytes(D), smem + L::kV + (value_block & 1) * L::kStage,
                      reinterpret_cast<float*>(smem + L::kValueScales + (value_block & 1) * L::kScaleBytes),
                      (from + value_block) * kTcKeys + token < longest,
                      std::true_type{});
        }
        fence_proxy_async_shared();
    };
    // ---- queries: half a row a thread, scaled by a power of two (exact) into
    // f16's range, in the codes' order.
    const int limit = row < live ? static_cast<int>(start + token_of(row) + 1) : 0;
    float* tops = reinterpret_cast<float*>(smem + L::kTops);
    std::uint32_t query_exponent;
    cp_async_wait_group<1>();
    __syncthreads();
    {
        uint4 raw[kUnits / 2];
        float most = 0.0f;
        bool bad = false;
#pragma unroll
        for (int u = 0; u < kUnits / 2; ++u) raw[u] = row < live ? *reinterpret_cast<const uint4*>(smem + query_at(row, half * (kUnits / 2) + u)) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < kUnits / 2; ++u) {
            float x[8];
            widen16(raw[u], x, QT{});
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                bad |= !isfinite(x[i]);
                most = fmaxf(most, fabsf(x[i]));
            }
        }
        if (bad) flag_error(p.error_word, kErrNonFinite);
        tops[threadIdx.x] = most;
        __syncthreads();
        most = fmaxf(tops[row], tops[row + kTcRows]);
        query_exponent = max(15u, __float_as_uint(most) >> 23);
        const float up = most > 0.0f ? __uint_as_float(min(254u, 268u - query_exponent) << 23) : 1.0f;
#pragma unroll
        for (int u = 0; u < kUnits / 2; ++u) {
            float x[8];
            widen16(raw[u], x, QT{});
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= up;
            *reinterpret_cast<uint4*>(smem + query_at(row, half * (kUnits / 2) + u)) =
                make_uint4(f16_pair(x[0], x[4]), f16_pair(x[1], x[5]), f16_pair(x[2], x[6]), f16_pair(x[3], x[7]));
        }
    }
    const float factor = p.scale_log2 * __uint_as_float((query_exponent - 14u) << 23);
    widen(0, kFirst);
    cp_async_wait_group<0>();
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    // The same in all lanes, and known to be.
    const std::uint32_t tmem = __shfl_sync(0xffffffffu, tmem_at, 0), at0 = __shfl_sync(0xffffffffu, at, 0);
    const bool issuer = __shfl_sync(0xffffffffu, warp, 0) == 0;
    const std::uint32_t my = tmem + (static_cast<std::uint32_t>((warp & 3) * 32) << 16);
    const tc::Waiter wait{&abort, p.error_word};
    // S of block b.
    auto scores = [&](int b) {
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
            const std::uint64_t q = tc::sw128_desc(at0 + L::kQ + k * L::kQGroup, 16, 1024);
            const std::uint64_t key = tc::sw128_desc(at0 + L::kK + (b & 1) * L::kStage + k * L::kKeyGroup, 16, 1024);
#pragma unroll
            for (int i = 0; i < 4; ++i) tc::mma_f16(tmem, q + 2 * i, key + 2 * i, tc::idesc_f16(0, 0, 0, kTcKeys), k > 0 || i > 0);
        }
        tc::mma_commit(&bars[kTcS]);
    };
    if (issuer && elect_one()) scores(0);
    widen(1, L::kRaw);
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars[kTcS]);

    const int clear = static_cast<int>(start + token_of(0) + 1);  // keys that all rows see
    float m = kNoScore;
    float2 l2 = make_float2(0.0f, 0.0f);
    for (int b = 0; b < blocks; ++b) {
        // ---- log2 scores of this half's 32 keys, two an instruction.
        float2 s[16];
        if (tc::warp_ok(wait(&bars[kTcS], b & 1))) {
            tc::tc_fence_after();
            std::uint32_t acc[2][16];
#pragma unroll
            for (int c = 0; c < 2; ++c) tmem_load16(my + 32 * half + 16 * c, acc[c]);
            const float4* units = reinterpret_cast<const float4*>(smem + L::kKeyScales + (b & 1) * L::kScaleBytes) + 8 * half;
#pragma unroll
            for (int c = 0; c < 2; ++c) tmem_wait16(acc[c]);
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float4 unit = units[i / 2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float2 sum = make_float2(__uint_as_float(acc[i / 8][2 * (i % 8 + j)]), __uint_as_float(acc[i / 8][2 * (i % 8 + j) + 1]));
                    s[i + j] = kv4::mul2(kv4::mul2(sum, j ? make_float2(unit.z, unit.w) : make_float2(unit.x, unit.y)), make_float2(factor, factor));
                }
            }
        }
        const int first = (from + b) * kTcKeys + 32 * half;
        if (first + 32 > clear) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (first + 2 * i >= limit) s[i].x = -INFINITY;
                if (first + 2 * i + 1 >= limit) s[i].y = -INFINITY;
            }
        }
        // ---- weights against m and in units of 2^e, from the rounded scores:
        // large scores differ from unrounded ones by more than the headroom.
        const float* units = reinterpret_cast<const float*>(smem + L::kValueScales + (b & 1) * L::kScaleBytes) + 32 * half;
        std::uint32_t weights[16];
        float2 sum;
        float most = 0.0f;
        auto weigh = [&] {
            sum = make_float2(0.0f, 0.0f);
            most = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float4 unit = *reinterpret_cast<const float4*>(units + 2 * i);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float2 w = make_float2(ex2_ftz(__fsub_rn(s[i + j].x, m)), ex2_ftz(__fsub_rn(s[i + j].y, m)));
                    sum = kv4::add2(sum, w);
                    const float2 scaled = kv4::mul2(w, j ? make_float2(unit.z, unit.w) : make_float2(unit.x, unit.y));
                    most = fmax3(most, scaled.x, scaled.y);
                    weights[i + j] = f16_pair(scaled.x, scaled.y);
                }
            }
        };
        if (b > 0) weigh();
        const bool rescale = __syncthreads_or(b == 0 || most > 32768.0f);
        if (*reinterpret_cast<volatile int*>(&abort)) break;  // set before the barrier only: the same for all
        fetch(at + L::kRaw);
        cp_async_commit();
        if (rescale) {
            float top = kNoScore;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float2 unit = *reinterpret_cast<const float2*>(units + 2 * i);
                top = fmax3(top, score_with_room(s[i].x, lg2(unit.x)), score_with_room(s[i].y, lg2(unit.y)));
            }
            tops[threadIdx.x] = top;
            __syncthreads();
            const float next = fmaxf(m, fmaxf(tops[row], tops[row + kTcRows])), alpha = ex2_ftz(m - next);
            m = next;
            l2 = kv4::mul2(l2, make_float2(alpha, alpha));
            if (b > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
                const std::uint32_t o_at = my + kTcKeys + half * (D / 2);
#pragma unroll 1
                for (int c = 0; c < D / 2; c += 16) {
                    std::uint32_t o[16];
                    tmem_load16(o_at + c, o);
                    tmem_wait16(o);
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                    tc::tmem_store16(o_at + c, o);
                }
            }
            weigh();
        }
        l2 = kv4::add2(l2, sum);
        tc::tmem_store16(my + 16 * half, weights);
        cp_async_wait_group<0>();
        tc::tmem_store_wait();
        tc::tc_fence_before();
        __syncthreads();  // the weights and the raw tiles are there
        if (issuer && elect_one()) {
            tc::tc_fence_after();
            // V is MN-major, 64 dims an atom.
            const std::uint64_t v = tc::sw128_desc(at0 + L::kV + (b & 1) * L::kStage, L::kKeyGroup, 1024);
#pragma unroll
            for (int i = 0; i < kTcKeys / 16; ++i) {
                tc::mma_f16_tmem_a(tmem + kTcKeys, tmem + 8 * i, v + 128 * i, tc::idesc_f16(0, 0, 1, D), b > 0 || i > 0);
            }
            if (b + 1 < blocks) scores(b + 1);
            else tc::mma_commit(&bars[kTcS]);
        }
        __syncwarp();
        widen(b + 2, L::kRaw);
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[kTcS]);
    }
    // ---- the row's output, or its sums for the merge; half of the dims a thread.
    if (!tc::warp_ok(wait(&bars[kTcS], blocks & 1))) l2 = make_float2(0.0f, 0.0f);
    tc::tc_fence_after();
    float* sums = reinterpret_cast<float*>(smem + L::kV);
    sums[threadIdx.x] = l2.x + l2.y;
    __syncthreads();
    const bool whole = splits == 1;
    {
        const float l = sums[row] + sums[row + kTcRows];
        const bool good = isfinite(l) && l > 0.0f;
        if (whole && !good && row < live) flag_error(p.error_word, kErrNormalizer);
        const float inv = !whole ? 1.0f : good ? 1.0f / l : 0.0f;
        // Through shared memory (over Q and K, 16-byte chunks swizzled by the row),
        // so that a row leaves in one piece; a split's sums are o [row][D], then
        // m and l per row (padded).
        float* part = p.ws_part + (static_cast<std::size_t>(work) * p.max_splits + split) * (kTcRows * (D + 4));
        if (!whole && half == 0) *reinterpret_cast<float2*>(part + kTcRows * D + 2 * row) = make_float2(m, l);
        auto staged = [&](int r, int chunk) { return reinterpret_cast<float4*>(smem + L::kQ + r * D * 4 + ((chunk ^ (r & 7)) << 4)); };
#pragma unroll
        for (int c0 = 0; c0 < D / 2; c0 += 16) {
            const int c1 = half * (D / 2) + c0;
            std::uint32_t o[16];
            tmem_load16(my + kTcKeys + c1, o);
            tmem_wait16(o);
#pragma unroll
            for (int u = 0; u < 16; u += 4) {
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(o[(u & 8) + 2 * i + (u >> 2 & 1)]) * inv;
                *staged(row, (c1 + u) / 4) = make_float4(x[0], x[1], x[2], x[3]);
            }
        }
        __syncthreads();
#pragma unroll 4
        for (int i = 0; i < D / 8; ++i) {
            const int own = copied_row(i, D / 4), r = 32 * (warp & 3) + own, chunk = lane % (D / 4);
            const std::size_t place = place_of(own);
            if (r >= live) continue;
            const float4 x = *staged(r, chunk);
            if (whole) store_row4(static_cast<QT*>(p.out) + place * D + 4 * chunk, x);
            else store_row4(part + r * D + 4 * chunk, x);
        }
    }
    if (threadIdx.x == 0) {
        // All MMAs are over before TMEM is released.
        tc::mma_commit(&bars[kTcDone]);
        mbar_wait_bounded(&bars[kTcDone], 0, p.error_word);
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, L::kTmem);
    }
    if (splits == 1) return;
    if (!last_of(p.ws_count + work, splits, ticket)) return;
    const float* parts = p.ws_part + static_cast<std::size_t>(work) * p.max_splits * (kTcRows * (D + 4));
    bool all_good = true;
#pragma unroll 2
    for (int i = threadIdx.x; i < live * D / 4; i += kTcThreads) {
        const int r = i / (D / 4);
        bool good;
        const float4 x = merge_parts<kTcRows * (D + 4), kTcRows * D>(parts, splits, r, i, good);
        all_good &= good;
        store_row4(static_cast<QT*>(p.out) + row_of(r) * D + 4 * i % D, x);
    }
    if (!all_good) flag_error(p.error_word, kErrNormalizer);
}

}  // namespace
}  // namespace ilb
