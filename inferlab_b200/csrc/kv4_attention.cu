// kv4_attention.cu - attention over a packed 4-bit pool (kv4.cuh): one decode
// step, and several query tokens per sequence.
//
// For a query q and the keys it sees, s_t = q . k_t / sqrt(D), p_t = exp(s_t -
// m), out = sum p_t v_t / sum p_t in one pass over the tokens with the running
// maximum m; k_t and v_t are the values the codes stand for.
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

struct Kv4Params {
    const unsigned char* arena;
    std::uint64_t num_blocks;
    std::uint32_t kv_heads, q_heads, tiles_per_block;
    const void* queries;
    void* out;
    const std::int32_t* tables;
    std::uint32_t max_blocks;
    long long max_context;
    const std::int32_t* context_lens;  // decode; null: segments
    const std::int32_t* starts;
    const std::int32_t* counts;
    const std::int32_t* offsets;
    std::uint32_t num_seqs;
    long long total_queries;
    float scale;
    std::uint32_t* error_word;
};

// One CTA per (query token, q-head): its D threads score D tokens at a time
// (one token each), then sum the value dim each owns.
template <typename RowT, typename QT, int D>
__global__ void __launch_bounds__(D) kv4_row_kernel(const Kv4Params p) {
    __shared__ float q_s[D], p_s[D], red[D / 32];
    __shared__ std::uint64_t tile_s[D / kv4::kTileTokens];
    const long long row = blockIdx.x / p.q_heads;
    const std::uint32_t head = blockIdx.x % p.q_heads;
    const std::uint32_t kv_head = head / (p.q_heads / p.kv_heads);
    QT* out = static_cast<QT*>(p.out) + (static_cast<std::size_t>(row) * p.q_heads + head) * D;

    long long seq = row, legal = 0;
    std::uint32_t error = 0;
    if (p.context_lens != nullptr) {
        legal = p.context_lens[row];
        if (legal < 0 || legal > p.max_context) error = kErrContext;
    } else {
        long long lo = 0, hi = static_cast<long long>(p.num_seqs) - 1;
        while (lo < hi) {
            const long long mid = (lo + hi + 1) >> 1;
            if (p.offsets[mid] <= row) lo = mid; else hi = mid - 1;
        }
        seq = lo;
        const long long index = row - p.offsets[lo], start = p.starts[lo], count = p.counts[lo];
        if (index < 0 || index >= count || start < 0 || start + count > p.max_context) error = kErrSegment;
        legal = start + index + 1;
    }
    if (error != 0 || legal == 0) {
        if (error != 0 && threadIdx.x == 0) flag_error(p.error_word, error);
        out[threadIdx.x] = Storage<QT>::from_float(0.0f);
        return;
    }
    const QT* q = static_cast<const QT*>(p.queries) + (static_cast<std::size_t>(row) * p.q_heads + head) * D;
    const float qv = Storage<RowT>::to_float(Storage<RowT>::from_float(Storage<QT>::to_float(q[threadIdx.x])));
    if (!isfinite(qv)) flag_error(p.error_word, kErrNonFinite);
    q_s[threadIdx.x] = qv;

    float m = -INFINITY, l = 0.0f, acc = 0.0f;
    const int slot = threadIdx.x % kv4::kTileTokens, tile_of = threadIdx.x / kv4::kTileTokens;
    for (long long t0 = 0; t0 < legal; t0 += D) {
        __syncthreads();
        const int n = static_cast<int>(min(static_cast<long long>(D), legal - t0));
        if (threadIdx.x < D / kv4::kTileTokens && threadIdx.x * kv4::kTileTokens < n) {
            const long long tile = t0 / kv4::kTileTokens + threadIdx.x;
            std::int32_t block = p.tables[static_cast<std::size_t>(seq) * p.max_blocks + tile / p.tiles_per_block];
            if (block < 0 || static_cast<std::uint64_t>(block) >= p.num_blocks) {
                flag_error(p.error_word, kErrBadBlock);
                block = 0;
            }
            tile_s[threadIdx.x] = ((static_cast<std::size_t>(block) * p.kv_heads + kv_head) * p.tiles_per_block +
                                   tile % p.tiles_per_block) * kv4::tile_bytes(D);
        }
        __syncthreads();
        float s = -INFINITY;
        if (threadIdx.x < n) {
            const unsigned char* tile = p.arena + tile_s[tile_of];
            s = 0.0f;
            for (int u = 0; u < D / 8; ++u) {
                const std::uint32_t word = *reinterpret_cast<const std::uint32_t*>(tile + kv4::key_word(D, slot, u));
                const float2 pair = kv4::load_pair(tile, kv4::pair_at(D, slot, u / 8, 0));
#pragma unroll
                for (int i = 0; i < 8; ++i) s = fmaf(q_s[8 * u + i], kv4::code_value(word, i, pair), s);
            }
            s *= p.scale;
        }
        float top = warp_max(s);
        if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = top;
        __syncthreads();
        for (int w = 0; w < D / 32; ++w) top = fmaxf(top, red[w]);
        const float next = fmaxf(m, top);
        const float alpha = m == -INFINITY ? 0.0f : expf(m - next);
        const float prob = s == -INFINITY ? 0.0f : expf(s - next);
        p_s[threadIdx.x] = prob;
        const float sum = warp_sum(prob);
        __syncthreads();
        if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = sum;
        __syncthreads();
        float tile_sum = 0.0f;
        for (int w = 0; w < D / 32; ++w) tile_sum += red[w];
        l = l * alpha + tile_sum;
        m = next;
        acc *= alpha;
        for (int t = 0; t < n; ++t) {
            const unsigned char* tile = p.arena + tile_s[t / kv4::kTileTokens];
            const int at = t % kv4::kTileTokens, u = static_cast<int>(threadIdx.x) / 8;
            const std::uint32_t word = *reinterpret_cast<const std::uint32_t*>(tile + kv4::value_word(D, at, u));
            acc = fmaf(p_s[t], kv4::code_value(word, threadIdx.x % 8, kv4::load_pair(tile, kv4::pair_at(D, at, u / 8, 1))), acc);
        }
    }
    out[threadIdx.x] = Storage<QT>::from_float(acc / l);
}

void check_kv4(const InferlabCudaKvPool& p, std::uint32_t query_dtype, std::uint32_t q_heads,
               std::uint32_t max_blocks, std::uint32_t max_context_len) {
    if (p.kv_bits != 4) throw std::runtime_error("4-bit attention needs a 4-bit pool");
    if (query_dtype != kFp32 && query_dtype != p.dtype) {
        throw std::runtime_error("4-bit attention query dtype must be FP32 or the pool's row type");
    }
    if (q_heads == 0 || q_heads % p.kv_heads != 0) {
        throw std::runtime_error("4-bit attention q_heads must be a positive multiple of kv_heads");
    }
    if (max_blocks == 0 || max_context_len == 0) {
        throw std::runtime_error("4-bit attention block table and context bound must be positive");
    }
}

void run_kv4(InferlabCudaKvPool& p, Kv4Params k, std::uint32_t query_dtype,
             std::uint32_t max_context_len, cudaStream_t s) {
    k.arena = static_cast<const unsigned char*>(p.key_arena);
    k.num_blocks = p.num_blocks;
    k.kv_heads = p.kv_heads;
    k.tiles_per_block = p.block_tokens / kv4::kTileTokens;
    k.max_context = std::min<long long>(max_context_len, static_cast<long long>(k.max_blocks) * p.block_tokens);
    k.scale = 1.0f / std::sqrt(static_cast<float>(p.head_dim));
    k.error_word = p.error_word;
    const std::uint64_t rows = static_cast<std::uint64_t>(k.total_queries) * k.q_heads;
    if (rows > 0x7FFFFFFFull) throw std::runtime_error("4-bit attention batch is too large");
    auto launch = [&](auto row_type, auto query_type) {
        using RowT = decltype(row_type);
        using QT = decltype(query_type);
        if (p.head_dim == 128) kv4_row_kernel<RowT, QT, 128><<<static_cast<unsigned>(rows), 128, 0, s>>>(k);
        else kv4_row_kernel<RowT, QT, 64><<<static_cast<unsigned>(rows), 64, 0, s>>>(k);
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
    if (pool == nullptr || pool->kv_bits != 4 || num_seqs == 0 || q_heads == 0 ||
        max_query_count == 0 || max_context_len == 0) {
        return 0;
    }
    return 0;
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
        check_kv4(p, query_dtype, q_heads, max_blocks_per_seq, max_context_len);
        DeviceGuard guard(p.device);
        Kv4Params k{};
        k.queries = queries;
        k.out = out;
        k.tables = block_tables;
        k.max_blocks = max_blocks_per_seq;
        k.context_lens = context_lens;
        k.num_seqs = num_seqs;
        k.total_queries = num_seqs;
        k.q_heads = q_heads;
        (void)workspace;
        (void)workspace_bytes;
        run_kv4(p, k, query_dtype, max_context_len, static_cast<cudaStream_t>(stream));
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
        check_kv4(p, query_dtype, q_heads, max_blocks_per_seq, max_context_len);
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
        k.num_seqs = num_segments;
        k.total_queries = static_cast<long long>(total_queries);
        k.q_heads = q_heads;
        (void)workspace;
        (void)workspace_bytes;
        run_kv4(p, k, query_dtype, max_context_len, static_cast<cudaStream_t>(stream));
    });
}
