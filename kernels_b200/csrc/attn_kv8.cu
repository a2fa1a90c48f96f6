// attn_kv8.cu -- attention of new tokens over the paged 8-bit key/value cache.
//
//   o = sum_j exp(scale q.k_j - lse) v_j,  lse = log(sum_j exp(scale q.k_j) [+ exp(sink)])
//   over keys j with p - window < j <= p, p the token's position
//
// One CTA per (token, query head): its warps take every fourth key with a
// running maximum and sum each, and are merged at the end.
#include "attn_few.cuh"

#include <algorithm>
#include <cmath>

using namespace graft;
using namespace graft::dev;

namespace {

__device__ unsigned g_attn_err;

template <int DT, int FMT>
__global__ void __launch_bounds__(128) attn_simple_kernel(const __grid_constant__ AttnArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ float sm[4], sl[4], so[4][256];
    const int t = blockIdx.x, h = blockIdx.y, hk = h / a.group;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int b = 0;
    for (uint32_t s0 = 1; s0 < a.n_seqs; s0 += blockDim.x) {
        const uint32_t s = s0 + threadIdx.x;
        b += __syncthreads_count(s < a.n_seqs && a.cu[s] <= t);
    }
    const int c0 = a.cu[b], n = a.cu[b + 1] - c0, start = a.start[b];
    if (t < c0 || t >= c0 + n) return;
    if (n > (int)a.max_tokens || (uint64_t)c0 + (uint64_t)n > a.tokens || start < 0 || (uint64_t)((int64_t)start + n) > a.max_len) {
        if (threadIdx.x == 0) atomicOr(&g_attn_err, (unsigned)GRAFT_KV_EBOUNDS);
        return;
    }
    const int p = start + t - c0, lo = a.window && p >= (int)a.window ? p - (int)a.window + 1 : 0;
    const int words = a.dim / 4;       // 4-byte words of a row; lane l has words l, l + 32
    float q[2][4], o[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int w = lane + 32 * i;
#pragma unroll
        for (int e = 0; e < 4; ++e) q[i][e] = o[i][e] = 0.f;
        if (w < words) {
            const uint2 x = *reinterpret_cast<const uint2*>((const uint16_t*)a.q + t * a.q_tok +
                                                            h * a.q_head + 4 * w);
            const float2 y = unpack2<DT>(x.x), z = unpack2<DT>(x.y);
            q[i][0] = y.x, q[i][1] = y.y, q[i][2] = z.x, q[i][3] = z.y;
        }
    }
    float m = -INFINITY, l = 0.f;
    for (int j = lo + warp; j <= p; j += 4) {
        const int blk = a.table[(size_t)b * a.table_stride + j / a.bt];
        if ((uint32_t)blk >= a.n_blocks) {
            if (lane == 0) atomicOr(&g_attn_err, (unsigned)GRAFT_KV_EBLOCK);
            continue;
        }
        const size_t bh = (size_t)blk * a.heads + hk, at = (bh * a.bt + j % a.bt) * a.dim;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (lane + 32 * i < words) {
                float f[4];
                kv_decode4<FMT>(*reinterpret_cast<const uint32_t*>(a.k + at + 4 * (lane + 32 * i)), f);
#pragma unroll
                for (int e = 0; e < 4; ++e) s = fmaf(f[e], q[i][e], s);
            }
        s = warp_sum(s) * a.k_scale[bh] * a.scale;
        const float mn = fmaxf(m, s), c = m == -INFINITY ? 0.f : exp2f((m - mn) * kLog2e);
        const float w = s == -INFINITY ? 0.f : exp2f((s - mn) * kLog2e);   // (a NaN stays one)
        m = mn;
        l = l * c + w;
        const float wv = w * a.v_scale[bh];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (lane + 32 * i < words) {
                float f[4];
                kv_decode4<FMT>(*reinterpret_cast<const uint32_t*>(a.v + at + 4 * (lane + 32 * i)), f);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][e] = fmaf(wv, f[e], o[i][e] * c);
            }
    }
    if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (lane + 32 * i < words)
#pragma unroll
            for (int e = 0; e < 4; ++e) so[warp][4 * (lane + 32 * i) + e] = o[i][e];
    __syncthreads();
    const float sink = a.sinks ? a.sinks[h] : -INFINITY;
    float M = sink;
    for (int w = 0; w < 4; ++w) M = fmaxf(M, sm[w]);
    float L = 0.f, f[4];
    for (int w = 0; w < 4; ++w) {
        f[w] = sl[w] == 0.f ? 0.f : exp2f((sm[w] - M) * kLog2e);
        L += f[w] * sl[w];
    }
    if (sink != -INFINITY) L += exp2f((sink - M) * kLog2e);
    for (int d = threadIdx.x; d < (int)a.dim; d += 128) {
        float v = 0.f;
        for (int w = 0; w < 4; ++w) v += f[w] * so[w][d];
        v = L != 0.f ? v / L : 0.f;
        uint16_t* y = (uint16_t*)a.out + t * a.o_tok + h * a.o_head + d;
        *y = (uint16_t)pack2<DT>(v, 0.f);
    }
    if (a.lse && threadIdx.x == 0)
        a.lse[(size_t)t * a.q_heads + h] = L != 0.f ? M + logf(L) : -INFINITY;
}

// ---- few query rows
template <int DP, int NT, int FMT, bool FULL>
int launch_few(AttnArgs a, cudaStream_t st) {
    DeviceInfo di;
    int rc = current_device_info(&di);
    if (rc) return rc;
    constexpr int smem = kFewSmem<DP, NT>;
    const auto kern = attn_few_kernel<DP, NT, FMT, FULL>;
    int per_sm = 1;
    if ((rc = ensure_smem((const void*)kern, smem)) ||
        (rc = occupancy((const void*)kern, kFewThreads, smem, &per_sm)))
        return rc;
    unsigned* err = nullptr;
    GRAFT_CUDA(cudaGetSymbolAddress((void**)&err, g_attn_err));
    // no more CTAs than the longest possible range has pieces
    const uint64_t keys = a.window ? std::min<uint64_t>(a.max_len, (uint64_t)a.window + a.max_tokens)
                                   : a.max_len;
    a.min_units = 2 * kFewWarps;
    a.pad_units = 2 * kFewWarps;
    const uint64_t units = keys / kFewUnit<DP> + 2 + a.pad_units;
    const uint64_t pairs = (uint64_t)a.n_seqs * a.heads;
    GRAFT_REQUIRE(pairs * units < (1ull << 31), "max_len %u of %u sequences is too long", a.max_len,
                  a.n_seqs);
    const uint64_t want = std::max(pairs, pairs * units / a.min_units + 1);
    const int grid = (int)std::min<uint64_t>(std::min(di.sm_count * per_sm, kAttnMaxGrid), want);
    return launch_pdl("attn_kv8", kern, dim3(grid), kFewThreads, smem, st, a, err);
}
template <int DP, int NT>
int launch_few(const AttnArgs& a, uint32_t fmt, cudaStream_t st) {
    if (a.dim == DP)
        return fmt == GRAFT_KV_INT8 ? launch_few<DP, NT, GRAFT_KV_INT8, true>(a, st)
                                    : launch_few<DP, NT, GRAFT_KV_E4M3, true>(a, st);
    return fmt == GRAFT_KV_INT8 ? launch_few<DP, NT, GRAFT_KV_INT8, false>(a, st)
                                : launch_few<DP, NT, GRAFT_KV_E4M3, false>(a, st);
}

// Query rows that the few-row kernel takes for a head_dim (registers).
int few_rows(uint32_t dim) { return dim <= 64 ? 32 : dim <= 128 ? 16 : 8; }

int check_attn(const GraftKVCache* cache, const GraftKVRange* range, const GraftAttnParams* P) {
    int rc;
    if ((rc = kv_check_cache(cache)) || (rc = kv_check_range(cache, range))) return rc;
    GRAFT_REQUIRE(P, "params pointer is null");
    GRAFT_REQUIRE(P->q_heads >= 1 && P->q_heads <= 32767 && P->q_heads % cache->kv_heads == 0,
                  "q_heads %u must be a multiple of kv_heads %u", P->q_heads, cache->kv_heads);
    GRAFT_REQUIRE(std::isfinite(P->scale), "scale must be finite");
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
    const size_t slot = d <= 64 ? kFewPartial<64, 4> : d <= 128 ? kFewPartial<128, 2>
                                                                : kFewPartial<256, 1>;
    return kAttnMaxGrid * (4 + 2 * 4 * slot);
}

extern "C" int graft_attn_kv8_init(void* ws, size_t ws_bytes, graft_stream_t stream) {
    clear_error();
    GRAFT_REQUIRE(ws && aligned(ws, 256), "the workspace must be 256-byte aligned");
    GRAFT_CUDA(cudaMemsetAsync(ws, 0, ws_bytes, stream));
    return GRAFT_OK;
}

extern "C" int graft_attn_kv8(const GraftKVCache* cache, const GraftHeads* q, const GraftHeads* out,
                              const GraftKVRange* range, const float* sinks, float* lse,
                              const GraftAttnParams* P, void* ws, size_t ws_bytes,
                              graft_stream_t stream) {
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
    a.q_heads = P->q_heads, a.group = P->q_heads / cache->kv_heads, a.window = P->window;
    a.scale = P->scale;
    a.bt_log2 = a.bt == 16 ? 4 : a.bt == 32 ? 5 : a.bt == 64 ? 6 : 7;
    a.bf16 = q->dtype == GRAFT_BF16;
    a.counters = (unsigned*)ws;
    a.partials = (float*)((char*)ws + kAttnMaxGrid * 4);
    const uint64_t rows = (uint64_t)range->max_tokens * a.group;
    if (range->max_tokens == 0) return GRAFT_OK;
    if (rows <= (uint64_t)few_rows(a.dim)) {
        if (a.dim <= 64)
            return rows <= 8    ? launch_few<64, 1>(a, cache->format, stream)
                   : rows <= 16 ? launch_few<64, 2>(a, cache->format, stream)
                                : launch_few<64, 4>(a, cache->format, stream);
        if (a.dim <= 128)
            return rows <= 8 ? launch_few<128, 1>(a, cache->format, stream)
                             : launch_few<128, 2>(a, cache->format, stream);
        return launch_few<256, 1>(a, cache->format, stream);
    }
    void (*kern)(const AttnArgs);
    if (q->dtype == GRAFT_F16)
        kern = cache->format == GRAFT_KV_INT8 ? attn_simple_kernel<GRAFT_F16, GRAFT_KV_INT8>
                                              : attn_simple_kernel<GRAFT_F16, GRAFT_KV_E4M3>;
    else
        kern = cache->format == GRAFT_KV_INT8 ? attn_simple_kernel<GRAFT_BF16, GRAFT_KV_INT8>
                                              : attn_simple_kernel<GRAFT_BF16, GRAFT_KV_E4M3>;
    return launch_pdl("attn_kv8", kern, dim3(q->tokens, P->q_heads), 128, 0, stream, a);
}
