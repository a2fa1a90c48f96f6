// attn_launch.cuh -- the launches of the attention kernels over the 8-bit cache.  Each file that
// includes this has kernels and an error word of its own.
#pragma once
#include "attn_chunk.cuh"
#include "attn_few.cuh"

#include <algorithm>
#include <atomic>

namespace graft {

// attn_tree.cu
int launch_attn_tree(const dev::AttnArgs& a, uint32_t format, uint64_t rows, cudaStream_t stream);
size_t attn_tree_partials(uint32_t dim, uint64_t rows);   // floats of a call's partial results, at most
unsigned attn_tree_device_errors(bool clear);

namespace {

using namespace dev;

__device__ unsigned g_attn_err;

// The error word's address on a device (asked for once).
int error_word(int device, unsigned** out) {
    static std::atomic<unsigned*> known[64];
    unsigned* p = device < 64 ? known[device].load(std::memory_order_relaxed) : nullptr;
    if (!p) {
        GRAFT_CUDA(cudaGetSymbolAddress((void**)&p, g_attn_err));
        if (device < 64) known[device].store(p, std::memory_order_relaxed);
    }
    *out = p;
    return GRAFT_OK;
}

// ---- few query rows
template <int DP, int NT, int FMT, bool FULL, bool TREE>
int launch_few(AttnArgs a, cudaStream_t st) {
    DeviceInfo di;
    int rc = current_device_info(&di);
    if (rc) return rc;
    constexpr int smem = kFewSmem<DP, NT>;
    const auto kern = attn_few_kernel<DP, NT, FMT, FULL, TREE>;
    int per_sm = 1;
    if ((rc = ensure_smem((const void*)kern, smem)) ||
        (rc = occupancy((const void*)kern, kFewThreads, smem, &per_sm)))
        return rc;
    unsigned* err = nullptr;
    if ((rc = error_word(di.device, &err))) return rc;
    // no more CTAs than the longest possible range has pieces
    const uint64_t keys = a.window ? std::min<uint64_t>(a.max_len, (uint64_t)a.window + a.max_tokens)
                                   : a.max_len;
    // A CTA's share is at least two units a warp, and a piece of a pair costs about three
    // more (queries, first copies, join): 32 sequences with windows of 128 keys take 27 us
    // without the pad and 9.8 with it, 64 of up to 8192 keys 122 and 102.
    a.min_units = 2 * kFewWarps;
    a.pad_units = 3 * kFewWarps;
    const uint64_t units = keys / kFewUnit<DP> + 2 + a.pad_units;
    const uint64_t pairs = (uint64_t)a.n_seqs * a.heads;
    // (units and a piece's edge beyond them are counted in 31 bits)
    GRAFT_REQUIRE(pairs * units < (1ull << 31) - a.pad_units - a.min_units,
                  "max_len %u of %u sequences is too long", a.max_len, a.n_seqs);
    const uint64_t want = std::max(2 * pairs, pairs * units / a.min_units + 1);
    const int grid = (int)std::min<uint64_t>(std::min(di.sm_count * per_sm, kAttnMaxGrid), want);
    return launch_pdl("attn_kv8", kern, dim3(grid), kFewThreads, smem, st, a, err);
}
template <int DP, int NT, bool TREE>
int launch_few(const AttnArgs& a, uint32_t fmt, cudaStream_t st) {
    if (a.dim == DP)
        return fmt == GRAFT_KV_INT8 ? launch_few<DP, NT, GRAFT_KV_INT8, true, TREE>(a, st)
                                    : launch_few<DP, NT, GRAFT_KV_E4M3, true, TREE>(a, st);
    return fmt == GRAFT_KV_INT8 ? launch_few<DP, NT, GRAFT_KV_INT8, false, TREE>(a, st)
                                : launch_few<DP, NT, GRAFT_KV_E4M3, false, TREE>(a, st);
}

// ---- many query rows
template <int DP, int FMT, bool TREE>
int launch_chunk(AttnArgs a, cudaStream_t st) {
    using C = Chunk<DP>;
    DeviceInfo di;
    int rc = current_device_info(&di);
    if (rc) return rc;
    const auto kern = attn_chunk_kernel<DP, FMT, TREE>;
    if ((rc = ensure_smem((const void*)kern, C::SMEM))) return rc;
    unsigned* err = nullptr;
    if ((rc = error_word(di.device, &err))) return rc;
    // a piece costs about as much besides its units as 3 units (queries in, output);
    // the pad is counted in keys
    a.min_units = 4;
    a.pad_units = 3 * C::KT;
    const uint64_t keys = a.window ? std::min<uint64_t>(a.max_len, (uint64_t)a.window + a.max_tokens)
                                   : a.max_len;
    const uint64_t units = keys / C::KT + 2;
    const uint64_t pairs = ((uint64_t)a.tokens / (C::ROWS / a.group) + a.n_seqs) * a.heads;
    GRAFT_REQUIRE(pairs < (1ull << 31) && (keys + a.pad_units) * a.heads < (1ull << 31),
                  "%u tokens, max_len %u are too many for one call", a.tokens, a.max_len);
    const uint64_t want = std::max(pairs, pairs * units / a.min_units + 1);
    const int grid = (int)std::min<uint64_t>(std::min(di.sm_count, kChunkMaxGrid), want);
    return launch_pdl("attn_kv8", kern, dim3(grid), C::THREADS, C::SMEM, st, a, err);
}
template <int DP, bool TREE>
int launch_chunk(const AttnArgs& a, uint32_t fmt, cudaStream_t st) {
    return fmt == GRAFT_KV_INT8 ? launch_chunk<DP, GRAFT_KV_INT8, TREE>(a, st)
                                : launch_chunk<DP, GRAFT_KV_E4M3, TREE>(a, st);
}

// Query rows that the few-row kernel takes for a head_dim (registers).
uint32_t few_rows(uint32_t dim) { return dim <= 64 ? 32 : dim <= 128 ? 16 : 8; }

template <bool TREE>
int launch_attn(const AttnArgs& a, uint32_t format, uint64_t rows, cudaStream_t stream) {
    if (rows <= few_rows(a.dim)) {
        if (a.dim <= 64)
            return rows <= 8    ? launch_few<64, 1, TREE>(a, format, stream)
                   : rows <= 16 ? launch_few<64, 2, TREE>(a, format, stream)
                                : launch_few<64, 4, TREE>(a, format, stream);
        if (a.dim <= 128)
            return rows <= 8 ? launch_few<128, 1, TREE>(a, format, stream)
                             : launch_few<128, 2, TREE>(a, format, stream);
        return launch_few<256, 1, TREE>(a, format, stream);
    }
    return a.dim <= 64    ? launch_chunk<64, TREE>(a, format, stream)
           : a.dim <= 128 ? launch_chunk<128, TREE>(a, format, stream)
                          : launch_chunk<256, TREE>(a, format, stream);
}

}  // namespace
}  // namespace graft
