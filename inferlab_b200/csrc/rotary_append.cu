// rotary_append.cu - token rows into the paged pool with the position rotation
// applied on the way, and rows read back.
//   K8 rotary_append_kernel: Q rows rotated to q_out; K rows rotated, V rows
//      as they are, rounded to the pool type (or quantised, kv4.cuh) and
//      written at (table[pos / block_tokens], pos % block_tokens).
//   K9 gather_rows_kernel: the rows at given (sequence, position) pairs, or of
//      one sequence's first tokens, as [rows][kv_heads][head_dim].
// The reference appends rows as the projection leaves them (PagedKvPool::append,
// worker/cpp/inferlab_runtime.cpp:713-767; its positions are learned vectors
// added to the hidden state) and has no quantised cache.
//
// Rotation of the pair (a, b) at a position with (cos, sin):
// (a cos - b sin, b cos + a sin), each product and sum rounded to fp32 once,
// then the result rounded once to the stored type. Pairs are (i, i + R / 2), or
// (2 i, 2 i + 1) when interleaved, over the first R = rotary_dim dims.
#include "common.cuh"
#include "internal.cuh"
#include "kv4.cuh"
#include "pool.cuh"

#include "../../include/inferlab_attention.h"

#include <algorithm>
#include <type_traits>

namespace ilb {
namespace {

struct AppendParams {
    const void* queries;
    const void* keys;
    const void* values;
    std::uint64_t q_stride, k_stride, v_stride;  // elements between token rows
    std::uint32_t q_heads, kv_heads, head_dim;
    const float* cos_sin;  // [positions][rotary_dim]: cosines, then sines
    std::uint64_t cos_sin_positions;  // no limit without rotation
    std::uint32_t rotary_dim;
    bool interleaved;
    bool padded_rows;  // sequence -1 is a padded row, not an error
    const std::int32_t* row_sequences;
    const std::int32_t* positions;
    const std::int32_t* tables;
    std::uint32_t num_seqs, max_blocks, block_tokens;
    std::uint64_t num_blocks;
    // Vector kernel: heads of a K/V round, Q items of a head and heads of a Q round; by_*
    // divide a thread number (< 256) as (t * by) >> 16.
    std::uint32_t heads, by_units, items, by_items, q_step;
    void* q_out;
    unsigned char* key_arena;  // 4-bit pools: the packed arena
    unsigned char* value_arena;
    std::uint32_t* error_word;
};

// Where a row goes: block id and slot, or -1 when the row is to be skipped
// (a padded row, sequence -1, without an error).
struct Place {
    std::int32_t block;
    std::uint32_t slot;
    std::int32_t position;
};

__device__ __forceinline__ Place find_place(std::int32_t seq, std::int32_t pos,
                                            const std::int32_t* tables, std::uint32_t num_seqs,
                                            std::uint32_t max_blocks, std::uint32_t block_tokens,
                                            std::uint64_t num_blocks, std::uint64_t positions,
                                            bool padded_rows, std::uint32_t& error) {
    error = 0;
    if (padded_rows && seq == -1) return Place{-1, 0, 0};
    if (seq < 0 || static_cast<std::uint32_t>(seq) >= num_seqs || pos < 0 ||
        static_cast<std::uint64_t>(pos) >= positions ||
        static_cast<std::uint32_t>(pos) / block_tokens >= max_blocks) {
        error = kErrPosition;
        return Place{-1, 0, 0};
    }
    const std::int32_t block = tables[static_cast<std::size_t>(seq) * max_blocks +
                                      static_cast<std::uint32_t>(pos) / block_tokens];
    if (block < 0 || static_cast<std::uint64_t>(block) >= num_blocks) {
        error = kErrBadBlock;
        return Place{-1, 0, 0};
    }
    return Place{block, static_cast<std::uint32_t>(pos) % block_tokens, pos};
}

// Dim d of a head's row, rotated. `angles`: the position's [rotary_dim] row.
template <typename RowT>
__device__ __forceinline__ float rotated(const RowT* head, std::uint32_t d, const float* angles,
                                         std::uint32_t rotary_dim, bool interleaved) {
    const float x = Storage<RowT>::to_float(head[d]);
    if (d >= rotary_dim) return x;
    const std::uint32_t half = rotary_dim / 2;
    const std::uint32_t pair = interleaved ? d / 2 : (d < half ? d : d - half);
    const bool first = interleaved ? d % 2 == 0 : d < half;
    const std::uint32_t other = interleaved ? (first ? d + 1 : d - 1) : (first ? d + half : d - half);
    const float y = Storage<RowT>::to_float(head[other]);
    const float c = angles[pair], s = angles[half + pair];
    return first ? __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s))
                 : __fadd_rn(__fmul_rn(x, c), __fmul_rn(y, s));
}

constexpr int kRowThreads = 256;

// Any shape: one CTA per token row, elements (8-dim units in a 4-bit pool)
// spread over its threads. K and V are checked before any of them is written,
// and the second pass finds them in L1; Q goes out either way.
template <typename RowT, typename PoolT, typename OutT, bool kFourBit>
__global__ void __launch_bounds__(kRowThreads) rotary_append_kernel(const AppendParams p) {
    const std::size_t row = blockIdx.x;
    std::uint32_t error = 0;
    const Place place = find_place(p.row_sequences[row], p.positions[row], p.tables, p.num_seqs,
                                   p.max_blocks, p.block_tokens, p.num_blocks, p.cos_sin_positions,
                                   p.padded_rows, error);
    if (error != 0 || place.block < 0) {
        if (error != 0 && threadIdx.x == 0) flag_error(p.error_word, error);
        return;
    }
    const float* angles = p.cos_sin + static_cast<std::size_t>(place.position) * p.rotary_dim;
    const RowT* key_row = static_cast<const RowT*>(p.keys) + row * p.k_stride;
    const RowT* value_row = static_cast<const RowT*>(p.values) + row * p.v_stride;
    const std::uint32_t d = p.head_dim;

    if constexpr (kFourBit) {
        const std::uint32_t per_head = d / 8;
        const std::uint32_t units = p.kv_heads * per_head;
        const std::size_t tile_size = kv4::tile_bytes(d);
        const std::size_t tiles_per_head = p.block_tokens / kv4::kTileTokens;
        unsigned char* tile0 = p.key_arena +
            (static_cast<std::size_t>(place.block) * p.kv_heads * tiles_per_head + place.slot / kv4::kTileTokens) * tile_size;
        const int slot = static_cast<int>(place.slot % kv4::kTileTokens);
        for (int pass = 0; pass < 2; ++pass) {
            bool any_bad = false;
            for (std::uint32_t first = 0; first < 2 * units; first += blockDim.x) {
                // Whole octets are live or not (units is a multiple of 8).
                const std::uint32_t at = first + threadIdx.x;
                const bool live = at < 2 * units;
                const bool is_value = live && at >= units;
                const std::uint32_t unit = live ? (is_value ? at - units : at) : 0;
                const std::uint32_t head = unit / per_head, u = unit % per_head;
                float x[8];
                const RowT* src = (is_value ? value_row : key_row) + static_cast<std::size_t>(head) * d;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float v = is_value ? Storage<RowT>::to_float(src[8 * u + i])
                                             : rotated(src, 8 * u + i, angles, p.rotary_dim, p.interleaved);
                    x[i] = Storage<PoolT>::to_float(Storage<PoolT>::from_float(v));
                }
                __half2 pair;
                bool bad;
                const std::uint32_t word = kv4::quantise(x, pair, bad);
                any_bad |= live && bad;
                if (pass == 1 && live) {
                    unsigned char* tile = tile0 + head * tiles_per_head * tile_size;
                    const int dd = static_cast<int>(d), uu = static_cast<int>(u);
                    *reinterpret_cast<std::uint32_t*>(
                        tile + (is_value ? kv4::value_word(dd, slot, uu) : kv4::key_word(dd, slot, uu))) = word;
                    if (u % 8 == 0) {
                        *reinterpret_cast<__half2*>(tile + kv4::pair_at(dd, slot, uu / 8, is_value)) = pair;
                    }
                }
            }
            if (pass == 0 && __syncthreads_or(any_bad)) {
                if (threadIdx.x == 0) flag_error(p.error_word, kErrNonFinite);
                break;
            }
        }
    } else {
        const std::size_t width = static_cast<std::size_t>(p.kv_heads) * d;
        bool bad = false;
        for (std::size_t i = threadIdx.x; i < width; i += blockDim.x) {
            const std::uint32_t head = i / d, dim = i % d;
            const float k = rotated(key_row + static_cast<std::size_t>(head) * d, dim, angles, p.rotary_dim, p.interleaved);
            bad |= !isfinite(Storage<PoolT>::to_float(Storage<PoolT>::from_float(k)));
            bad |= !isfinite(Storage<PoolT>::to_float(Storage<PoolT>::from_float(Storage<RowT>::to_float(value_row[i]))));
        }
        const bool rejected = __syncthreads_or(bad);
        if (rejected && threadIdx.x == 0) flag_error(p.error_word, kErrNonFinite);
        for (std::size_t i = threadIdx.x; i < width && !rejected; i += blockDim.x) {
            const std::uint32_t head = i / d, dim = i % d;
            const std::size_t dst =
                ((static_cast<std::size_t>(place.block) * p.kv_heads + head) * p.block_tokens + place.slot) * d + dim;
            const float k = rotated(key_row + static_cast<std::size_t>(head) * d, dim, angles, p.rotary_dim, p.interleaved);
            reinterpret_cast<PoolT*>(p.key_arena)[dst] = Storage<PoolT>::from_float(k);
            reinterpret_cast<PoolT*>(p.value_arena)[dst] = Storage<PoolT>::from_float(Storage<RowT>::to_float(value_row[i]));
        }
    }
    if (p.queries != nullptr) {
        const RowT* q_row = static_cast<const RowT*>(p.queries) + row * p.q_stride;
        const std::size_t width = static_cast<std::size_t>(p.q_heads) * d;
        OutT* out = static_cast<OutT*>(p.q_out) + row * width;
        for (std::size_t i = threadIdx.x; i < width; i += blockDim.x) {
            out[i] = Storage<OutT>::from_float(rotated(q_row + i / d * d, static_cast<std::uint32_t>(i % d), angles,
                                                       p.rotary_dim, p.interleaved));
        }
    }
}

// Eight consecutive elements as fp32, 16 bytes a load.
template <typename T>
__device__ __forceinline__ void load8(const T* at, float (&x)[8]) {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int c = 0; c < 8 / kPer; ++c) widen16(reinterpret_cast<const uint4*>(at)[c], &x[c * kPer], T{});
}
template <typename T>
struct Eight {
    uint4 words[8 * sizeof(T) / 16];
};
__device__ __forceinline__ std::uint32_t round_pair(float low, float high, __half) {
    const __half2 v = __floats2half2_rn(low, high);
    return *reinterpret_cast<const std::uint32_t*>(&v);
}
__device__ __forceinline__ std::uint32_t round_pair(float low, float high, __nv_bfloat16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(low, high);
    return *reinterpret_cast<const std::uint32_t*>(&v);
}
// Rounded to T.
template <typename T>
__device__ __forceinline__ Eight<T> round8(const float (&x)[8]) {
    Eight<T> e;
    if constexpr (sizeof(T) == 4) {
        e.words[0] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
        e.words[1] = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7]));
    } else {
        e.words[0] = make_uint4(round_pair(x[0], x[1], T{}), round_pair(x[2], x[3], T{}), round_pair(x[4], x[5], T{}),
                                round_pair(x[6], x[7], T{}));
    }
    return e;
}
// Whether a value rounds to something T cannot hold as a finite number (a NaN
// compares false): from half a unit above T's largest.
template <typename T>
__device__ __forceinline__ bool outside8(const float (&x)[8]) {
    const float limit = sizeof(T) == 4 ? INFINITY : std::is_same<T, __half>::value ? 65520.0f : __uint_as_float(0x7f7f8000u);
    bool out = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) out |= !(fabsf(x[i]) < limit);
    return out;
}
template <typename T>
__device__ __forceinline__ Eight<T> ask8(const T* at) {
    Eight<T> e;
#pragma unroll
    for (int c = 0; c < static_cast<int>(8 * sizeof(T) / 16); ++c) e.words[c] = reinterpret_cast<const uint4*>(at)[c];
    return e;
}
template <typename T>
__device__ __forceinline__ void store8(T* at, const Eight<T>& e) {
#pragma unroll
    for (int c = 0; c < static_cast<int>(8 * sizeof(T) / 16); ++c) reinterpret_cast<uint4*>(at)[c] = e.words[c];
}

// One half of split pairs, y the other: x c - y s, or (second) x c + y s, each
// product and sum rounded once, products two lanes a time.
__device__ __forceinline__ void turn8(float (&x)[8], const float (&y)[8], const float (&c)[8], const float (&s)[8],
                                      bool second) {
    const std::uint32_t sign = second ? 0u : 0x80000000u;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float2 own = kv4::mul2(make_float2(x[i], x[i + 1]), make_float2(c[i], c[i + 1]));
        const float2 other = kv4::mul2(make_float2(y[i], y[i + 1]), make_float2(s[i], s[i + 1]));
        x[i] = __fadd_rn(own.x, __uint_as_float(__float_as_uint(other.x) ^ sign));
        x[i + 1] = __fadd_rn(own.y, __uint_as_float(__float_as_uint(other.y) ^ sign));
    }
}
// Interleaved: c and s hold four angles, the pairs are neighbours.
__device__ __forceinline__ void turn8_neighbours(float (&x)[8], const float (&c)[8], const float (&s)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = x[2 * i], b = x[2 * i + 1];
        x[2 * i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
        x[2 * i + 1] = __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, s[i]));
    }
}

// Four consecutive elements.
template <typename T>
struct Four {
    std::uint32_t words[sizeof(T)];
};
template <typename T>
__device__ __forceinline__ Four<T> ask4(const T* at) {
    Four<T> e;
    if constexpr (sizeof(T) == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(at);
        e.words[0] = x.x, e.words[1] = x.y, e.words[2] = x.z, e.words[3] = x.w;
    } else {
        const uint2 x = *reinterpret_cast<const uint2*>(at);
        e.words[0] = x.x, e.words[1] = x.y;
    }
    return e;
}
template <typename T>
__device__ __forceinline__ void widen4(const Four<T>& e, float (&x)[4]) {
    const T* t = reinterpret_cast<const T*>(e.words);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = Storage<T>::to_float(t[i]);
}
template <typename T>
__device__ __forceinline__ void store4(T* at, const float (&x)[4]) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(at) = make_float4(x[0], x[1], x[2], x[3]);
    else *reinterpret_cast<uint2*>(at) = make_uint2(round_pair(x[0], x[1], T{}), round_pair(x[2], x[3], T{}));
}

// The common shapes: units of 8 dims, 16-byte accesses, two CTAs per row.
//   K and V (blockIdx.y 0): a thread keeps to one unit of the head and goes
//     through the heads, p.heads at a time, in at most kPasses rounds, held
//     until the whole row is known to be good; in a 4-bit pool eight neighbours
//     then hold a group. The partner dims of a split rotation are loaded a
//     second time (from L1).
//   Q (blockIdx.y 1): a thread takes four dims and their partners, so nothing is
//     loaded or widened twice, and asks for several heads' at once.
// Everything of a row is asked for in one round of loads behind its sequence and
// position, and what it is short of is rows in flight: 8192 rows of 16 + 16 + 16
// fp32 heads x 128 into an f16 pool take 57 us (90% of the copy rate), of 32 + 8 +
// 8 bf16 heads into 4 bits, 12 KB in and 8 + 2.3 KB out each, 51 (28 at that
// rate; 59% of the issue slots and a third of DRAM used, warps wait for their
// rows). As one CTA of 256 threads and 64 registers, or with Q by eight dims (70
// registers), a tenth more.
template <typename RowT, typename PoolT, typename OutT, bool kFourBit, bool kNeighbours, int kPasses>
__global__ void __launch_bounds__(kRowThreads) rotary_append_vector_kernel(const AppendParams p) {
    const std::size_t row = blockIdx.x;
    const std::uint32_t d = p.head_dim, half = p.rotary_dim / 2;
    const std::int32_t seq = p.row_sequences[row], position = p.positions[row];
    std::uint32_t error = 0;
    auto find = [&] {
        return find_place(seq, position, p.tables, p.num_seqs, p.max_blocks, p.block_tokens, p.num_blocks,
                          p.cos_sin_positions, p.padded_rows, error);
    };
    // A position behind the table is found out with the place; it is not read.
    const bool known = position >= 0 && static_cast<std::uint64_t>(position) < p.cos_sin_positions;
    const float* angles = p.cos_sin + static_cast<std::size_t>(position) * p.rotary_dim;

    if (blockIdx.y != 0) {
        // A Q item is four dims and their partners, or four that do not turn
        // (neighbours: four dims, their own partners).
        const std::uint32_t turning = kNeighbours ? p.rotary_dim / 4 : p.rotary_dim / 8;
        std::uint32_t h = (threadIdx.x * p.by_items) >> 16;
        const std::uint32_t item = threadIdx.x - h * p.items, step = p.q_step;
        if (h >= step || h >= p.q_heads) return;  // left over
        const bool turns = item < turning;
        const std::uint32_t dim = turns ? 4 * item : p.rotary_dim + 4 * (item - turning);
        const RowT* q_row = static_cast<const RowT*>(p.queries) + row * p.q_stride + dim;
        // Heads asked for at once: 16 bits want the registers (48 us, 2 heads 51),
        // fp32 the loads (55 us, 2 heads 58).
        constexpr int kRounds = sizeof(RowT) == 4 ? 4 : 1;
        Four<RowT> q1[kRounds], q2[kRounds];
        auto ask = [&] {
#pragma unroll
            for (int i = 0; i < kRounds; ++i) {
                if (h + i * step >= p.q_heads) break;
                const RowT* at = q_row + static_cast<std::size_t>(h + i * step) * d;
                q1[i] = ask4(at);
                if (!kNeighbours && turns) q2[i] = ask4(at + half);
            }
        };
        ask();
        float c[4], s[4];
        if (turns && known) {
            if constexpr (kNeighbours) {
                const float2 x = *reinterpret_cast<const float2*>(angles + 2 * item);
                const float2 y = *reinterpret_cast<const float2*>(angles + half + 2 * item);
                c[0] = x.x, c[1] = x.y, s[0] = y.x, s[1] = y.y;
            } else {
                widen16(*reinterpret_cast<const uint4*>(angles + 4 * item), c, 0.0f);
                widen16(*reinterpret_cast<const uint4*>(angles + half + 4 * item), s, 0.0f);
            }
        }
        if (find().block < 0) return;  // a bad row is reported by the other CTA
        OutT* out_row = static_cast<OutT*>(p.q_out) + row * p.q_heads * d + dim;
        for (;;) {
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                if (h + r * step >= p.q_heads) return;
                float a[4], b[4];
                widen4(q1[r], a);
                if (!kNeighbours && turns) widen4(q2[r], b);
                OutT* out = out_row + static_cast<std::size_t>(h + r * step) * d;
                if (turns) {
                    if constexpr (kNeighbours) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float x = a[2 * i], y = a[2 * i + 1];
                            a[2 * i] = __fsub_rn(__fmul_rn(x, c[i]), __fmul_rn(y, s[i]));
                            a[2 * i + 1] = __fadd_rn(__fmul_rn(y, c[i]), __fmul_rn(x, s[i]));
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i += 2) {
                            const float2 x = make_float2(a[i], a[i + 1]), y = make_float2(b[i], b[i + 1]);
                            const float2 cc = make_float2(c[i], c[i + 1]), ss = make_float2(s[i], s[i + 1]);
                            const float2 xc = kv4::mul2(x, cc), ys = kv4::mul2(y, ss), yc = kv4::mul2(y, cc), xs = kv4::mul2(x, ss);
                            a[i] = __fsub_rn(xc.x, ys.x), a[i + 1] = __fsub_rn(xc.y, ys.y);
                            b[i] = __fadd_rn(yc.x, xs.x), b[i + 1] = __fadd_rn(yc.y, xs.y);
                        }
                        store4(out + half, b);
                    }
                }
                store4(out, a);
            }
            h += kRounds * step;
            ask();
        }
    }

    const std::uint32_t units = d / 8, heads = p.heads;
    const std::uint32_t h0 = (threadIdx.x * p.by_units) >> 16, u = threadIdx.x - h0 * units;
    const RowT* key_row = static_cast<const RowT*>(p.keys) + row * p.k_stride + 8 * u;
    const RowT* value_row = static_cast<const RowT*>(p.values) + row * p.v_stride + 8 * u;
    const bool turns = 8 * u < p.rotary_dim, second = !kNeighbours && 8 * u >= half;
    const int partner = second ? -static_cast<int>(half) : static_cast<int>(half);
    // Rounds in which this warp has a head (a quantising warp works whole).
    const std::uint32_t warp_h0 = ((threadIdx.x & ~31u) * p.by_units) >> 16;
    auto has = [&](int i) { return warp_h0 + i * heads < p.kv_heads; };
    Eight<RowT> k_in[kPasses], k2_in[kPasses], v_in[kPasses];
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        if (!has(i)) break;
        const std::uint32_t h = min(h0 + i * heads, p.kv_heads - 1);
        k_in[i] = ask8(key_row + static_cast<std::size_t>(h) * d);
        if (!kNeighbours && turns) k2_in[i] = ask8(key_row + static_cast<std::size_t>(h) * d + partner);
        v_in[i] = ask8(value_row + static_cast<std::size_t>(h) * d);
    }
    float c[8], s[8];
    if (turns && known) {
        if constexpr (kNeighbours) {
            widen16(*reinterpret_cast<const uint4*>(angles + 4 * u), c, 0.0f);
            widen16(*reinterpret_cast<const uint4*>(angles + half + 4 * u), s, 0.0f);
        } else {
            load8(angles + (second ? 8 * u - half : 8 * u), c);
            load8(angles + (second ? 8 * u : 8 * u + half), s);
        }
    }
    const Place place = find();
    if (error != 0 || place.block < 0) {
        if (error != 0 && threadIdx.x == 0) flag_error(p.error_word, error);
        return;
    }
    float k[kPasses][8], v[kPasses][8];
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        if (!has(i)) break;
        load8(reinterpret_cast<const RowT*>(k_in[i].words), k[i]);
        load8(reinterpret_cast<const RowT*>(v_in[i].words), v[i]);
        if (!turns) continue;
        if constexpr (kNeighbours) {
            turn8_neighbours(k[i], c, s);
        } else {
            float other[8];
            load8(reinterpret_cast<const RowT*>(k2_in[i].words), other);
            turn8(k[i], other, c, s, second);
        }
    }

    bool bad = false;
    if constexpr (kFourBit) {
        std::uint32_t words[kPasses][2];
        __half2 pairs[kPasses][2];
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            if (!has(i)) break;
            const bool live = h0 + i * heads < p.kv_heads;
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                float (&x)[8] = which ? v[i] : k[i];
                bool out_of_range;
                const Eight<PoolT> rounded = round8<PoolT>(x);
                widen16(rounded.words[0], x, PoolT{});
                words[i][which] = kv4::quantise(x, pairs[i][which], out_of_range);
                bad |= live && out_of_range;
            }
        }
        if (__syncthreads_or(bad)) {
            if (threadIdx.x == 0) flag_error(p.error_word, kErrNonFinite);
            return;
        }
        const std::size_t tiles_per_head = p.block_tokens / kv4::kTileTokens;
        const int slot = static_cast<int>(place.slot % kv4::kTileTokens), uu = static_cast<int>(u);
        auto write = [&](auto dim) {  // head_dim as a constant
            constexpr int kD = decltype(dim)::value;
            unsigned char* tile0 = p.key_arena +
                (static_cast<std::size_t>(place.block) * p.kv_heads * tiles_per_head + place.slot / kv4::kTileTokens) * kv4::tile_bytes(kD);
#pragma unroll
            for (int i = 0; i < kPasses; ++i) {
                const std::uint32_t h = h0 + i * heads;
                if (h >= p.kv_heads) break;
                unsigned char* tile = tile0 + h * tiles_per_head * kv4::tile_bytes(kD);
                *reinterpret_cast<std::uint32_t*>(tile + kv4::key_word(kD, slot, uu)) = words[i][0];
                *reinterpret_cast<std::uint32_t*>(tile + kv4::value_word(kD, slot, uu)) = words[i][1];
                if (u % 8 < 2) {
                    *reinterpret_cast<__half2*>(tile + kv4::pair_at(kD, slot, uu / 8, uu % 8)) = uu % 8 == 0 ? pairs[i][0] : pairs[i][1];
                }
            }
        };
        if (d == 128) write(std::integral_constant<int, 128>{});
        else write(std::integral_constant<int, 64>{});
    } else {
        Eight<PoolT> held[kPasses][2];
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            if (!has(i)) break;
            bad |= outside8<PoolT>(k[i]) || outside8<PoolT>(v[i]);
            held[i][0] = round8<PoolT>(k[i]);
            held[i][1] = round8<PoolT>(v[i]);
        }
        if (__syncthreads_or(bad)) {
            if (threadIdx.x == 0) flag_error(p.error_word, kErrNonFinite);
            return;
        }
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const std::uint32_t h = h0 + i * heads;
            if (h >= p.kv_heads) break;
            const std::size_t dst =
                ((static_cast<std::size_t>(place.block) * p.kv_heads + h) * p.block_tokens + place.slot) * d + 8 * u;
            store8(reinterpret_cast<PoolT*>(p.key_arena) + dst, held[i][0]);
            store8(reinterpret_cast<PoolT*>(p.value_arena) + dst, held[i][1]);
        }
    }
}

struct GatherParams {
    const unsigned char* key_arena;
    const unsigned char* value_arena;
    const std::int32_t* row_sequences;  // null: sequence 0, position = row
    const std::int32_t* positions;
    const std::int32_t* tables;
    std::uint32_t num_seqs, max_blocks, block_tokens, kv_heads, head_dim;
    std::uint64_t num_blocks;
    void* keys_out;
    void* values_out;
    std::uint32_t* error_word;
};

// The common shapes of a gather: units of 8 dims, 16-byte accesses; a 4-bit
// pool's unit is one word of codes and its group's pair. Bound by a short CTA's
// chain of loads (place, table, tile): 8192 rows of 8 + 8 heads x 128 of a 4-bit
// pool 14 us (7 at the copy rate; 256 threads a row a quarter more), of 16 + 16
// heads of an f16 pool 28 (20).
constexpr int kGatherThreads = 128;
template <typename T, bool kFourBit>
__global__ void __launch_bounds__(kGatherThreads) gather_rows_vector_kernel(const GatherParams p) {
    const std::size_t row = blockIdx.x;
    std::uint32_t error = 0;
    const Place place = find_place(p.row_sequences != nullptr ? p.row_sequences[row] : 0,
                                   p.positions != nullptr ? p.positions[row] : static_cast<std::int32_t>(row),
                                   p.tables, p.num_seqs, p.max_blocks, p.block_tokens, p.num_blocks,
                                   ~0ull, p.row_sequences != nullptr, error);
    if (place.block < 0) {
        if (error != 0 && threadIdx.x == 0) flag_error(p.error_word, error);
        return;
    }
    const std::uint32_t units = p.head_dim / 8, all = p.kv_heads * units;
    for (std::uint32_t i = threadIdx.x; i < 2 * all; i += blockDim.x) {
        const bool is_value = i >= all;
        const std::uint32_t unit = is_value ? i - all : i;
        // A 4-bit pool's heads are 8 or 16 units: a shift.
        const std::uint32_t head = kFourBit ? unit >> (units == 16 ? 4 : 3) : unit / units, u = unit - head * units;
        T* out = static_cast<T*>(is_value ? p.values_out : p.keys_out) + (row * all + unit) * 8;
        if constexpr (kFourBit) {
            const std::uint32_t tiles_per_head = p.block_tokens / kv4::kTileTokens;
            const int slot = static_cast<int>(place.slot % kv4::kTileTokens), uu = static_cast<int>(u);
            auto widen = [&](auto dim) {  // head_dim as a constant
                constexpr int kD = decltype(dim)::value;
                const unsigned char* tile = p.key_arena +
                    ((static_cast<std::size_t>(place.block) * p.kv_heads + head) * tiles_per_head +
                     place.slot / kv4::kTileTokens) * kv4::tile_bytes(kD);
                const std::uint32_t word = *reinterpret_cast<const std::uint32_t*>(
                    tile + (is_value ? kv4::value_word(kD, slot, uu) : kv4::key_word(kD, slot, uu)));
                float x[8];
                kv4::code_values(word, kv4::load_pair(tile, kv4::pair_at(kD, slot, uu / 8, is_value)), x);
                if (std::is_same<T, __half>::value) {  // bf16 holds all of them: at most 9 x 65504
#pragma unroll
                    for (int n = 0; n < 8; ++n) x[n] = fminf(fmaxf(x[n], -65504.0f), 65504.0f);
                }
                store8(out, round8<T>(x));
            };
            if (p.head_dim == 128) widen(std::integral_constant<int, 128>{});
            else widen(std::integral_constant<int, 64>{});
        } else {
            const T* at = reinterpret_cast<const T*>(is_value ? p.value_arena : p.key_arena) +
                ((static_cast<std::size_t>(place.block) * p.kv_heads + head) * p.block_tokens + place.slot) * p.head_dim + 8 * u;
            Eight<T> e;
#pragma unroll
            for (int c = 0; c < static_cast<int>(8 * sizeof(T) / 16); ++c) e.words[c] = reinterpret_cast<const uint4*>(at)[c];
            store8(out, e);
        }
    }
}

// Any shape, one CTA per row. Words of the pool's own element type are copied bit for
// bit; a 4-bit pool's codes are widened and rounded to its row type T,
// saturating at T's largest finite value.
template <typename T, bool kFourBit>
__global__ void __launch_bounds__(kRowThreads) gather_rows_kernel(const GatherParams p) {
    const std::size_t row = blockIdx.x;
    std::uint32_t error = 0;
    const Place place = find_place(p.row_sequences != nullptr ? p.row_sequences[row] : 0,
                                   p.positions != nullptr ? p.positions[row] : static_cast<std::int32_t>(row),
                                   p.tables, p.num_seqs, p.max_blocks, p.block_tokens, p.num_blocks,
                                   ~0ull, p.row_sequences != nullptr, error);
    if (place.block < 0) {
        if (error != 0 && threadIdx.x == 0) flag_error(p.error_word, error);
        return;
    }
    const std::uint32_t d = p.head_dim;
    const std::size_t width = static_cast<std::size_t>(p.kv_heads) * d;
    T* keys = static_cast<T*>(p.keys_out) + row * width;
    T* values = static_cast<T*>(p.values_out) + row * width;
    if constexpr (kFourBit) {
        const float most = std::is_same<T, __half>::value ? 65504.0f : 3.3895313892515355e38f;
        const std::size_t tiles_per_head = p.block_tokens / kv4::kTileTokens;
        const int slot = static_cast<int>(place.slot % kv4::kTileTokens);
        for (std::size_t i = threadIdx.x; i < 2 * width / 8; i += blockDim.x) {
            const bool is_value = i >= width / 8;
            const std::size_t unit = is_value ? i - width / 8 : i;
            const std::size_t head = unit / (d / 8);
            const int u = static_cast<int>(unit % (d / 8)), dd = static_cast<int>(d);
            const unsigned char* tile = p.key_arena +
                ((static_cast<std::size_t>(place.block) * p.kv_heads + head) * tiles_per_head +
                 place.slot / kv4::kTileTokens) * kv4::tile_bytes(dd);
            const std::uint32_t word = *reinterpret_cast<const std::uint32_t*>(
                tile + (is_value ? kv4::value_word(dd, slot, u) : kv4::key_word(dd, slot, u)));
            const float2 pair = kv4::load_pair(tile, kv4::pair_at(dd, slot, u / 8, is_value));
            T* out = (is_value ? values : keys) + unit * 8;
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                out[n] = Storage<T>::from_float(fminf(fmaxf(kv4::code_value(word, n, pair), -most), most));
            }
        }
    } else {
        for (std::size_t i = threadIdx.x; i < width; i += blockDim.x) {
            const std::size_t src =
                ((static_cast<std::size_t>(place.block) * p.kv_heads + i / d) * p.block_tokens + place.slot) * d + i % d;
            keys[i] = reinterpret_cast<const T*>(p.key_arena)[src];
            values[i] = reinterpret_cast<const T*>(p.value_arena)[src];
        }
    }
}

template <typename RowT, typename PoolT, typename OutT, bool kFourBit>
void launch_vector(const AppendParams& a, unsigned grid, unsigned threads, std::uint32_t passes, cudaStream_t s) {
    auto launch = [&](auto neighbours) {
        constexpr bool kN = decltype(neighbours)::value;
        auto* kernel = passes == 1 ? rotary_append_vector_kernel<RowT, PoolT, OutT, kFourBit, kN, 1>
                     : passes == 2 ? rotary_append_vector_kernel<RowT, PoolT, OutT, kFourBit, kN, 2>
                                   : rotary_append_vector_kernel<RowT, PoolT, OutT, kFourBit, kN, 4>;
        kernel<<<dim3(grid, a.queries != nullptr ? 2 : 1), threads, 0, s>>>(a);
    };
    if (a.interleaved) launch(std::true_type{});
    else launch(std::false_type{});
}

bool aligned16(const void* at) { return reinterpret_cast<std::uintptr_t>(at) % 16 == 0; }

template <typename RowT, typename PoolT, typename OutT>
void launch_rotary(const AppendParams& a, std::uint64_t rows, bool four_bit, cudaStream_t s) {
    const unsigned grid = static_cast<unsigned>(rows);
    // The vector kernel's conditions: whole 8-dim units whose partners are whole
    // units too, every access on 16 bytes, and the row's K/V heads within four
    // rounds of the CTA (32 heads x 128 need two).
    const std::uint32_t units = a.head_dim / 8;
    const std::uint64_t step = 16 / sizeof(RowT);
    if (a.head_dim % 8 == 0 && units <= kRowThreads && a.rotary_dim % (a.interleaved ? 8 : 16) == 0 &&
        aligned16(a.keys) && aligned16(a.values) && a.k_stride % step == 0 && a.v_stride % step == 0 &&
        (a.queries == nullptr || (aligned16(a.queries) && aligned16(a.q_out) && a.q_stride % step == 0)) &&
        (a.rotary_dim == 0 || aligned16(a.cos_sin))) {
        // 128 threads, or 256 where they would need more than two K/V rounds or a
        // Q item each (8192 rows of 16 fp32 heads: 57 us, 256 threads 63).
        const std::uint32_t items = a.rotary_dim / (a.interleaved ? 4 : 8) + (a.head_dim - a.rotary_dim) / 4;
        const std::uint32_t wish = std::max(1u, 128 / units);
        std::uint32_t heads = a.kv_heads <= 2 * wish && items <= wish * units ? wish : kRowThreads / units;
        while (four_bit && heads * units % 32 != 0) ++heads;  // whole warps: the groups' minima are shuffled
        const std::uint32_t passes = (a.kv_heads + heads - 1) / heads;
        if (passes <= 4 && items <= heads * units) {
            AppendParams v = a;
            v.heads = heads;
            v.by_units = (65536 + units - 1) / units;
            v.items = items;
            v.by_items = (65536 + items - 1) / items;
            v.q_step = heads * units / items;
            if constexpr (!std::is_same<PoolT, float>::value) {
                if (four_bit) {
                    launch_vector<RowT, PoolT, OutT, true>(v, grid, heads * units, passes, s);
                    return;
                }
            }
            launch_vector<RowT, PoolT, OutT, false>(v, grid, heads * units, passes, s);
            return;
        }
    }
    if constexpr (!std::is_same<PoolT, float>::value) {
        if (four_bit) {
            rotary_append_kernel<RowT, PoolT, OutT, true><<<grid, kRowThreads, 0, s>>>(a);
            return;
        }
    }
    rotary_append_kernel<RowT, PoolT, OutT, false><<<grid, kRowThreads, 0, s>>>(a);
}

template <typename PoolT>
void select_rotary(const AppendParams& a, std::uint64_t rows, std::uint32_t row_dtype,
                   std::uint32_t out_dtype, bool four_bit, cudaStream_t s) {
    if constexpr (std::is_same<PoolT, float>::value) {
        launch_rotary<float, float, float>(a, rows, false, s);
    } else if (row_dtype == kFp32) {
        if (out_dtype == kFp32) launch_rotary<float, PoolT, float>(a, rows, four_bit, s);
        else launch_rotary<float, PoolT, PoolT>(a, rows, four_bit, s);
    } else {
        if (out_dtype == kFp32) launch_rotary<PoolT, PoolT, float>(a, rows, four_bit, s);
        else launch_rotary<PoolT, PoolT, PoolT>(a, rows, four_bit, s);
    }
}

void run_gather_rows(InferlabCudaKvPool& p, const std::int32_t* row_sequences,
                     const std::int32_t* positions, std::uint64_t rows, const std::int32_t* tables,
                     std::uint32_t num_seqs, std::uint32_t max_blocks, void* keys_out,
                     void* values_out, cudaStream_t s) {
    GatherParams g{};
    g.key_arena = static_cast<const unsigned char*>(p.key_arena);
    g.value_arena = static_cast<const unsigned char*>(p.value_arena);
    g.row_sequences = row_sequences;
    g.positions = positions;
    g.tables = tables;
    g.num_seqs = num_seqs;
    g.max_blocks = max_blocks;
    g.block_tokens = p.block_tokens;
    g.kv_heads = p.kv_heads;
    g.head_dim = p.head_dim;
    g.num_blocks = p.num_blocks;
    g.keys_out = keys_out;
    g.values_out = values_out;
    g.error_word = p.error_word;
    const unsigned grid = static_cast<unsigned>(rows);
    const bool whole = p.head_dim % 8 == 0 && aligned16(keys_out) && aligned16(values_out) &&
                       static_cast<std::uint64_t>(p.kv_heads) * p.head_dim < 0x7FFFFFFFull;
    auto launch = [&](auto type) {
        using T = decltype(type);
        if constexpr (!std::is_same<T, float>::value) {
            if (p.kv_bits != 0) {
                auto* kernel = whole ? gather_rows_vector_kernel<T, true> : gather_rows_kernel<T, true>;
                kernel<<<grid, whole ? kGatherThreads : kRowThreads, 0, s>>>(g);
                return;
            }
        }
        auto* kernel = whole ? gather_rows_vector_kernel<T, false> : gather_rows_kernel<T, false>;
        kernel<<<grid, whole ? kGatherThreads : kRowThreads, 0, s>>>(g);
    };
    if (p.dtype == kFp32) launch(float{});
    else if (p.dtype == kF16) launch(__half{});
    else launch(__nv_bfloat16{});
    cuda_check(cudaGetLastError(), "gather rows launch");
}

bool overlaps(const void* a, std::size_t a_bytes, const void* b, std::size_t b_bytes) {
    const auto a0 = reinterpret_cast<std::uintptr_t>(a), b0 = reinterpret_cast<std::uintptr_t>(b);
    return a0 < b0 + b_bytes && b0 < a0 + a_bytes;
}

}  // namespace

void launch_rotary_append(InferlabCudaKvPool& p, const InferlabCudaRotaryAppend& c,
                          bool padded_rows, cudaStream_t stream) {
    AppendParams a{};
    a.queries = c.q_heads != 0 ? c.queries : nullptr;
    a.keys = c.key_rows;
    a.values = c.value_rows;
    a.q_stride = c.query_stride;
    a.k_stride = c.key_stride;
    a.v_stride = c.value_stride;
    a.q_heads = c.q_heads;
    a.kv_heads = p.kv_heads;
    a.head_dim = p.head_dim;
    a.cos_sin = c.cos_sin;
    a.cos_sin_positions = c.rotary_dim != 0 ? c.cos_sin_positions : ~0ull;
    a.rotary_dim = c.rotary_dim;
    a.interleaved = c.interleaved != 0;
    a.padded_rows = padded_rows;
    a.row_sequences = c.row_sequences;
    a.positions = c.positions;
    a.tables = c.block_tables;
    a.num_seqs = c.num_seqs;
    a.max_blocks = c.max_blocks_per_seq;
    a.block_tokens = p.block_tokens;
    a.num_blocks = p.num_blocks;
    a.q_out = c.q_out;
    a.key_arena = static_cast<unsigned char*>(p.key_arena);
    a.value_arena = static_cast<unsigned char*>(p.value_arena);
    a.error_word = p.error_word;
    const bool four_bit = p.kv_bits != 0;
    if (p.dtype == kFp32) {
        select_rotary<float>(a, c.rows, c.row_dtype, c.q_out_dtype, four_bit, stream);
    } else if (p.dtype == kF16) {
        select_rotary<__half>(a, c.rows, c.row_dtype, c.q_out_dtype, four_bit, stream);
    } else {
        select_rotary<__nv_bfloat16>(a, c.rows, c.row_dtype, c.q_out_dtype, four_bit, stream);
    }
    cuda_check(cudaGetLastError(), "rotary append launch");
}

void launch_kv4_gather(InferlabCudaKvPool& p, const std::int32_t* block_table, std::uint64_t tokens,
                       void* keys_out, void* values_out, cudaStream_t stream) {
    const std::uint32_t blocks = static_cast<std::uint32_t>((tokens + p.block_tokens - 1) / p.block_tokens);
    run_gather_rows(p, nullptr, nullptr, tokens, block_table, 1, blocks, keys_out, values_out, stream);
}

}  // namespace ilb

extern "C" int inferlab_cuda_kv_append_rotary(InferlabCudaKvPool* pool,
                                              const InferlabCudaRotaryAppend* call, void* stream,
                                              char* error, std::size_t error_capacity) {
    return ilb::protect(error, error_capacity, [&] {
        using namespace ilb;
        auto& p = checked_pool(pool);
        if (call == nullptr) throw std::runtime_error("rotary append description is null");
        const InferlabCudaRotaryAppend& c = *call;
        if (c.rows == 0) return;
        if (c.key_rows == nullptr || c.value_rows == nullptr || c.row_sequences == nullptr ||
            c.positions == nullptr || c.block_tables == nullptr ||
            (c.q_heads != 0 && (c.queries == nullptr || c.q_out == nullptr)) ||
            (c.rotary_dim != 0 && c.cos_sin == nullptr)) {
            throw std::runtime_error("rotary append pointer is null");
        }
        if (c.row_dtype != kFp32 && c.row_dtype != p.dtype) {
            throw std::runtime_error("paged KV row dtype must be FP32 or the pool dtype");
        }
        if (c.q_heads != 0 && c.q_out_dtype != kFp32 && c.q_out_dtype != p.dtype) {
            throw std::runtime_error("rotary append query output dtype must be FP32 or the pool dtype");
        }
        if (c.rotary_dim % 2 != 0 || c.rotary_dim > p.head_dim) {
            throw std::runtime_error("rotary_dim must be even and at most head_dim");
        }
        if (c.num_seqs == 0 || c.max_blocks_per_seq == 0) throw std::runtime_error("paged KV block table is empty");
        if (c.rows > 0x7FFFFFFFull) throw std::runtime_error("paged KV append row count is too large");
        const std::uint64_t kv_width = static_cast<std::uint64_t>(p.kv_heads) * p.head_dim;
        const std::uint64_t q_width = static_cast<std::uint64_t>(c.q_heads) * p.head_dim;
        if (kv_width > 0x7FFFFFFFull || q_width > 0x7FFFFFFFull) throw std::runtime_error("rotary append rows are too wide");
        if (c.q_heads != 0) {
            // A dim's rotation reads its partner dim, which another thread may
            // already have replaced if the output were the input.
            const std::size_t in = c.row_dtype == kFp32 ? 4 : 2, out = c.q_out_dtype == kFp32 ? 4 : 2;
            const std::size_t out_bytes = checked_mul(checked_mul(c.rows, q_width, "rotary append is too large"), out,
                                                      "rotary append is too large");
            const auto span = [&](std::uint64_t stride, std::uint64_t width) {
                return (checked_mul(c.rows - 1, stride, "rotary append is too large") + width) * in;
            };
            if (overlaps(c.q_out, out_bytes, c.queries, span(c.query_stride, q_width)) ||
                overlaps(c.q_out, out_bytes, c.key_rows, span(c.key_stride, kv_width)) ||
                overlaps(c.q_out, out_bytes, c.value_rows, span(c.value_stride, kv_width))) {
                throw std::runtime_error("rotary append query output overlaps its input rows");
            }
        }
        DeviceGuard guard(p.device);
        launch_rotary_append(p, c, true, static_cast<cudaStream_t>(stream));
    });
}

extern "C" int inferlab_cuda_kv_gather_rows(InferlabCudaKvPool* pool, const std::int32_t* row_sequences,
                                            const std::int32_t* positions, std::uint64_t rows,
                                            const std::int32_t* block_tables, std::uint32_t num_seqs,
                                            std::uint32_t max_blocks_per_seq, void* keys_out,
                                            void* values_out, void* stream, char* error,
                                            std::size_t error_capacity) {
    return ilb::protect(error, error_capacity, [&] {
        using namespace ilb;
        auto& p = checked_pool(pool);
        if (rows == 0) return;
        if (row_sequences == nullptr || positions == nullptr || block_tables == nullptr ||
            keys_out == nullptr || values_out == nullptr) {
            throw std::runtime_error("paged KV gather pointer is null");
        }
        if (num_seqs == 0 || max_blocks_per_seq == 0) throw std::runtime_error("paged KV block table is empty");
        if (rows > 0x7FFFFFFFull) throw std::runtime_error("paged KV gather is too long");
        DeviceGuard guard(p.device);
        run_gather_rows(p, row_sequences, positions, rows, block_tables, num_seqs, max_blocks_per_seq,
                        keys_out, values_out, static_cast<cudaStream_t>(stream));
    });
}
