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
#include "attn_launch.cuh"

#include <cmath>

using namespace graft;
using namespace graft::dev;

namespace {

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
unsigned attn_device_errors(bool clear) {
    return read_device_errors(g_attn_err, clear) | attn_tree_device_errors(clear);
}
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
    // (trees take the same workspace, and may have their rows as columns)
    const uint64_t rows = (uint64_t)range->max_tokens * (P->q_heads / cache->kv_heads);
    return kAttnMaxGrid * 4 + 2 * 4 * std::max(floats, attn_tree_partials(d, rows));
}

extern "C" int graft_attn_kv8_init(void* ws, size_t ws_bytes, graft_stream_t stream) {
    clear_error();
    GRAFT_REQUIRE(ws && aligned(ws, 256), "the workspace must be 256-byte aligned");
    GRAFT_CUDA(cudaMemsetAsync(ws, 0, ws_bytes, stream));
    return GRAFT_OK;
}

namespace {

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
    return mask ? launch_attn_tree(a, cache->format, rows, stream)
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
    // (a step without new tokens may have no mask: empty buffers have no address)
    if (range->n_seqs && range->max_tokens && !(q && q->tokens == 0)) {
        GRAFT_REQUIRE(mask && aligned(mask, 4), "mask must be a 4-byte aligned buffer");
        GRAFT_REQUIRE(mask_stride >= (range->max_tokens + 31ull) / 32 || (q && q->tokens <= 1),
                      "mask_stride %llu does not hold max_tokens %u", (unsigned long long)mask_stride,
                      range->max_tokens);
        GRAFT_REQUIRE(P->window == 0 || (positions && aligned(positions, 4)),
                      "positions must be a 4-byte aligned buffer when there is a window");
    }
    return attend(cache, q, out, range, mask, mask_stride, positions, sinks, lse, P, ws, ws_bytes, stream);
}
