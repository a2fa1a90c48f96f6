// attn_kv8.cu -- attention of new tokens over the paged 8-bit key/value cache.
//
//   o = sum_j exp(scale q.k_j - lse) v_j,  lse = log(sum_j exp(scale q.k_j) [+ exp(sink)])
//   over keys j with p - window < j <= p, p the token's position
//
// Up to few_rows() query rows (tokens of a sequence x query heads of a key/value
// head) go to the kernel of attn_few.cuh, whose registers hold all of them: one
// pass over the keys at the rate of HBM.  More rows go to the kernel of
// attn_chunk.cuh (tcgen05), whose tiles have 128 rows whether they are full or not.
// Both sides of the rule, in us (64 query heads on 8 of 64; 32 on 8 of 128; 16 on 8 of 256):
//   131071 keys, 8 rows 38 | 153, 32 rows 67 | 154
//   32 sequences of up to 8192 keys, 8 rows 41 | 146, 16 rows 52 | 146, 32 rows 76 | 148
//   the same, heads of 128: 4 rows 57 | 200, 16 rows 92 | 204;  of 256: 8 rows 104 | 374
#include "attn_chunk.cuh"
#include "attn_few.cuh"

#include <algorithm>
#include <atomic>
#include <cmath>

using namespace graft;
using namespace graft::dev;

namespace {

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

int check_attn(const GraftKVCache* cache, const GraftKVRange* range, const GraftAttnParams* P) {
    int rc;
    if ((rc = kv_check_cache(cache)) || (rc = kv_check_range(cache, range))) return rc;
    GRAFT_REQUIRE(P, "params pointer is null");
    GRAFT_REQUIRE(P->q_heads >= 1 && P->q_heads <= 32767 && P->q_heads % cache->kv_heads == 0,
                  "q_heads %u must be a multiple of kv_heads %u", P->q_heads, cache->kv_heads);
    GRAFT_REQUIRE(P->q_heads / cache->kv_heads <= (cache->head_dim <= 128 ? 256u : 128u),
                  "%u query heads a key/value head are too many", P->q_heads / cache->kv_heads);
    GRAFT_REQUIRE(std::isfinite(P->scale), "scale must be finite");
    GRAFT_REQUIRE(range->n_seqs == 0 || range->max_len <= (1u << 30), "max_len %u out of range",
                  range->max_len);
    GRAFT_REQUIRE(P->window <= 0x7FFFFFFFu, "window %u out of range", P->window);
    return GRAFT_OK;
}

}  // namespace

namespace graft {
unsigned attn_device_errors(bool clear) { return read_device_errors(g_attn_err, clear); }
}  // namespace graft

extern "C" size_t graft_attn_kv8_workspace(const GraftKVCache* cache, const GraftKVRange* range,
                                           const GraftAttnParams* P) {
    if (check_attn(cache, range, P)) return 0;
    const uint32_t d = cache->head_dim;
    const bool few = (uint64_t)range->max_tokens * (P->q_heads / cache->kv_heads) <= few_rows(d);
    const size_t floats =
        few ? kAttnMaxGrid * (size_t)(d <= 64    ? kFewPartial<64, 4>
                                      : d <= 128 ? kFewPartial<128, 2> : kFewPartial<256, 1>)
            : kChunkMaxGrid * (size_t)(d <= 64    ? Chunk<64>::PARTIAL
                                       : d <= 128 ? Chunk<128>::PARTIAL : Chunk<256>::PARTIAL);
    return kAttnMaxGrid * 4 + 2 * 4 * floats;
}

extern "C" int graft_attn_kv8_init(void* ws, size_t ws_bytes, graft_stream_t stream) {
    clear_error();
    GRAFT_REQUIRE(ws && aligned(ws, 256), "the workspace must be 256-byte aligned");
    GRAFT_CUDA(cudaMemsetAsync(ws, 0, ws_bytes, stream));
    return GRAFT_OK;
}

namespace {

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

// mask: of a tree of new tokens, or null
int attend(const GraftKVCache* cache, const GraftHeads* q, const GraftHeads* out,
           const GraftKVRange* range, const int32_t* mask, uint64_t mask_stride,
           const int32_t* positions, const float* sinks, float* lse, const GraftAttnParams* P,
           void* ws, size_t ws_bytes, cudaStream_t stream) {
    int rc;
    if ((rc = check_attn(cache, range, P)) || (rc = kv_check_heads("q", q, cache->head_dim)) ||
        (rc = kv_check_heads("out", out, cache->head_dim)))
        return rc;
    GRAFT_REQUIRE(q->dtype == out->dtype && q->dtype != GRAFT_F32,
                  "q and out must both be fp16 or both bf16");
    GRAFT_REQUIRE(q->tokens == out->tokens, "q and out must have the same number of tokens");
    GRAFT_REQUIRE(aligned(sinks, 4) && aligned(lse, 4), "sinks and lse must be 4-byte aligned");
    const size_t need = graft_attn_kv8_workspace(cache, range, P);
    GRAFT_REQUIRE(ws && aligned(ws, 256) && ws_bytes >= need,
                  "the workspace must be 256-byte aligned and hold %zu bytes", need);
    if (range->n_seqs == 0 || q->tokens == 0) return GRAFT_OK;
    AttnArgs a = {};
    a.k = (const uint8_t*)cache->k, a.v = (const uint8_t*)cache->v;
    a.k_scale = cache->k_scale, a.v_scale = cache->v_scale;
    a.table = range->block_table, a.start = range->start, a.cu = range->cu_tokens;
    a.q = q->data, a.out = out->data, a.sinks = sinks, a.lse = lse;
    a.q_tok = q->token_stride, a.q_head = q->head_stride;
    a.o_tok = out->token_stride, a.o_head = out->head_stride;
    a.n_blocks = cache->n_blocks, a.heads = cache->kv_heads, a.bt = cache->block_tokens;
    a.dim = cache->head_dim, a.n_seqs = range->n_seqs, a.table_stride = range->table_stride;
    a.max_tokens = range->max_tokens, a.max_len = range->max_len, a.tokens = q->tokens;
    a.q_heads = P->q_heads, a.group = P->q_heads / cache->kv_heads;
    // (a window that reaches beyond every sequence, the largest int say, is none)
    a.window = P->window < range->max_len ? P->window : 0;
    a.scale = P->scale;
    a.bt_log2 = a.bt == 16 ? 4 : a.bt == 32 ? 5 : a.bt == 64 ? 6 : 7;
    a.bf16 = q->dtype == GRAFT_BF16;
    a.counters = (unsigned*)ws;
    a.partials = (float*)((char*)ws + kAttnMaxGrid * 4);
    const uint64_t rows = (uint64_t)range->max_tokens * a.group;
    if (range->max_tokens == 0) return GRAFT_OK;
    a.mask = (const uint32_t*)mask, a.mask_stride = mask_stride, a.positions = positions;
    return mask ? launch_attn<true>(a, cache->format, rows, stream)
                : launch_attn<false>(a, cache->format, rows, stream);
}

}  // namespace

extern "C" int graft_attn_kv8(const GraftKVCache* cache, const GraftHeads* q, const GraftHeads* out,
                              const GraftKVRange* range, const float* sinks, float* lse,
                              const GraftAttnParams* P, void* ws, size_t ws_bytes,
                              graft_stream_t stream) {
    return attend(cache, q, out, range, nullptr, 0, nullptr, sinks, lse, P, ws, ws_bytes, stream);
}

extern "C" int graft_attn_tree_kv8(const GraftKVCache* cache, const GraftHeads* q,
                                   const GraftHeads* out, const GraftKVRange* range,
                                   const int32_t* mask, uint64_t mask_stride,
                                   const int32_t* positions, const float* sinks, float* lse,
                                   const GraftAttnParams* P, void* ws, size_t ws_bytes,
                                   graft_stream_t stream) {
    int rc;
    if ((rc = check_attn(cache, range, P))) return rc;
    if (range->n_seqs && range->max_tokens) {
        GRAFT_REQUIRE(mask && aligned(mask, 4), "mask must be a 4-byte aligned buffer");
        GRAFT_REQUIRE(mask_stride >= (range->max_tokens + 31ull) / 32 || (q && q->tokens <= 1),
                      "mask_stride %llu does not hold max_tokens %u", (unsigned long long)mask_stride,
                      range->max_tokens);
        GRAFT_REQUIRE(P->window == 0 || (positions && aligned(positions, 4)),
                      "positions must be a 4-byte aligned buffer when there is a window");
    }
    return attend(cache, q, out, range, mask, mask_stride, positions, sinks, lse, P, ws, ws_bytes, stream);
}
