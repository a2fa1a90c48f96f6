// logprobs.cu -- log probability of a given token, entropy and the top
// alternatives of each row of logits, in one pass over the logits.
//
//   z = scale*logit, lse = log sum exp z, logprob = z[target] - lse,
//   entropy = lse - sum p z
//
// A row is cut into segments (few rows: to use the SMs; many: to balance
// them), a CTA takes one.  Each thread sums e = 2^d and e*d over its chunks of
// 16 bytes, d = (x - ref) scale log2(e), against a reference of its own that moves
// only when a logit passes it by 2^64: no maximum is needed first.  So
//   lse = scale*ref + ln L,  entropy = ln L - ln2 E / L      (L = sum e, E = sum e d)
// and HBM bounds a long call (one exponential an element keeps the MUFU at about
// 70% at that rate for 16-bit logits).
//
// The top k come from the threads' own maxima, which the pass finds on the
// way: the k-th largest of them bounds the k-th largest logit from below, so only
// the k threads whose maximum reaches it can hold one of the top k.  Their
// chunks (k / 256 of the segment) are read again, from L2, what reaches the
// bound is collected and ranked by counting.  Ties go to the lowest index: keys
// are (value, index) pairs, all different.  Segments meet in the workspace, and a
// row's last CTA joins them.
#include "kv_common.cuh"

#include <algorithm>
#include <cmath>

using namespace graft;
using namespace graft::dev;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxTop = 32, kMaxSegs = 16;
constexpr int kCap = 512;            // collected keys; more take the slow selection
constexpr int kMinSeg = 8192;        // elements of a segment, at least
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kRounds = 148 * 16;    // CTAs that fill the SMs for several rounds (148 x 4 x 4)
constexpr size_t kCounterBytes = (kRounds * 4 + 255) / 256 * 256;   // a row is cut only if rows < kRounds
constexpr uint64_t kNoKey = 0;       // below every key of a logit that is not -inf

struct Partial {                     // of a segment
    float ref, L, E, pad;
    uint64_t key[kMaxTop];
};

struct LpArgs {
    const void* logits;
    const int32_t* targets;
    float *logprob, *entropy, *top_lp;
    int32_t* top_idx;
    uint64_t row_stride;
    uint32_t rows, vocab, top_k;
    int segs;                        // of a row
    float scale;
    unsigned* counters;              // per row, zero between calls
    Partial* partials;               // [rows][segs]
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {   // a NaN stays one
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// fp32 in the order of unsigned integers (finite and infinite; -0 = +0)
__device__ __forceinline__ uint32_t order(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float unorder(uint32_t o) {
    return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) {
    return ((uint64_t)order(x) << 32) | (0xFFFFFFFFu - index);
}

template <int DT>
__device__ __forceinline__ float logit(const void* row, uint32_t i) {
    if constexpr (DT == GRAFT_F32) return ((const float*)row)[i];
    const uint16_t w = ((const uint16_t*)row)[i];
    return DT == GRAFT_F16 ? h2f(w) : bf2f(w);
}
template <int DT>
constexpr int kPer = DT == GRAFT_F32 ? 4 : 8;   // elements of a chunk

// Chunk c of a row whose first element is `off` elements into the row's first
// 16-byte chunk; elements outside the row are -inf and are not read.
template <int DT>
__device__ __forceinline__ uint4 load_chunk(const void* row, int off, uint32_t vocab, int c) {
    constexpr int N = kPer<DT>;
    const int first = c * N - off;
    if (first >= 0 && first + N <= (int)vocab)
        return ld_stream((const char*)row + (int64_t)first * (16 / N));
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == GRAFT_F32) {
            const int e = first + i;
            w[i] = e >= 0 && e < (int)vocab ? ((const uint32_t*)row)[e] : 0xFF800000u;
        } else {
            const uint32_t none = DT == GRAFT_F16 ? 0xFC00u : 0xFF80u;
            const int e = first + 2 * i;
            w[i] = (e >= 0 && e < (int)vocab ? ((const uint16_t*)row)[e] : none) |
                   (e + 1 >= 0 && e + 1 < (int)vocab ? ((const uint16_t*)row)[e + 1] : none) << 16;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <int DT>
__device__ __forceinline__ void floats_of(const uint4& v, float (&x)[kPer<DT>]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == GRAFT_F32) {
            x[i] = __uint_as_float(w[i]);
        } else {
            const float2 p = unpack2<DT>(w[i]);
            x[2 * i] = p.x, x[2 * i + 1] = p.y;
        }
    }
}

// (ref, L, E) of two parts; ref = -inf marks an empty one.  L and E are
// relative to their part's ref, c = scale log2(e).
__device__ __forceinline__ void join(float& ref, float& L, float& E, float r2, float L2, float E2,
                                     float c) {
    const float m = fmaxf(ref, r2);
    // (m - m is 0 or, for +inf, NaN, as it should be)
    const float a = ref == -INFINITY ? 0.f : (ref - m) * c, b = r2 == -INFINITY ? 0.f : (r2 - m) * c;
    const float fa = ref == -INFINITY ? 0.f : ex2(a), fb = r2 == -INFINITY ? 0.f : ex2(b);
    // (a part 2^126 below the other is 0, and 0 * -inf must not be NaN)
    E = fa * fmaf(L, max_nan(a, -256.f), E) + fb * fmaf(L2, max_nan(b, -256.f), E2);
    L = fa * L + fb * L2;
    ref = m;
}

struct Shared {
    float ref[kWarps], L[kWarps], E[kWarps];
    uint64_t key[kCap];
    uint64_t best[kMaxTop];
    uint64_t red[kWarps];
    int list[kMaxTop];
    int n, listed, last, count[2];
};

// Largest key below `limit` that `mine` yields over the CTA.
__device__ __forceinline__ uint64_t block_max(Shared& sh, uint64_t v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const uint64_t w = __shfl_xor_sync(~0u, v, o);
        v = w > v ? w : v;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.red[threadIdx.x >> 5] = v;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) v = sh.red[w] > v ? sh.red[w] : v;
    return v;
}

// Ranks the n different keys sh.key[0..n): sh.best[r] = the r-th largest, r < k.
__device__ __forceinline__ void rank_keys(Shared& sh, int n, int k) {
    for (int i = threadIdx.x; i < k; i += kThreads) sh.best[i] = kNoKey;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const uint64_t v = sh.key[i];
        int r = 0;
        for (int j = 0; j < n; ++j) r += sh.key[j] > v;
        if (r < k) sh.best[r] = v;
    }
    __syncthreads();
}

// The top k keys of the segment's chunks [c0, c1) into sh.best.  tmax, tchunk: the
// thread's largest logit (-inf: none) and the first chunk that holds it.
template <int DT>
__device__ __forceinline__ void select_top(Shared& sh, const void* row, int off, uint32_t vocab,
                                           int c0, int c1, float tmax, int tchunk, int k) {
    constexpr int N = kPer<DT>;
    const int tid = threadIdx.x;
    // ---- the k-th largest thread maximum, bit by bit (16-bit logits as fp32 differ in
    // their upper 16 or 19 bits only)
    constexpr int kLow = DT == GRAFT_F32 ? 0 : DT == GRAFT_BF16 ? 16 : 13;
    const bool some = tmax > -INFINITY;
    const uint32_t mine = some ? order(tmax) >> kLow : 0;
    uint32_t bound = 0;
    if (tid == 0) sh.n = sh.listed = 0;
    if (__syncthreads_count(some) > k) {
#pragma unroll 1
        for (int b = 31 - kLow; b >= 0; --b) {
            const uint32_t t = bound | (1u << b);
            if (__syncthreads_count(mine >= t) >= k) bound = t;
        }
    }
    bound = max(bound, 1u);
    // ---- equal maxima: the first chunks go first
    int last_chunk = 0x7FFFFFFF;
    const int above = __syncthreads_count(mine > bound);
    if (__syncthreads_count(mine >= bound) > k) {
        last_chunk = 0;
#pragma unroll 1
        for (int b = 30; b >= 0; --b) {   // the least t with k threads at or before it, minus 1
            const int t = last_chunk | (1 << b);
            if (above + __syncthreads_count(mine == bound && tchunk < t) < k) last_chunk = t;
        }
    }
    if (mine > bound || (mine == bound && tchunk <= last_chunk)) sh.list[atomicAdd(&sh.listed, 1)] = tid;
    __syncthreads();
    // ---- what reaches the bound in those threads' chunks
    const int listed = sh.listed, per = (c1 - c0 + kThreads - 1) / kThreads;
    for (int i = tid; i < listed * per; i += kThreads) {
        const int q = i / per, c = c0 + sh.list[q] + (i - q * per) * kThreads;
        if (c >= c1) continue;
        float x[N];
        floats_of<DT>(load_chunk<DT>(row, off, vocab, c), x);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const uint32_t o = x[e] > -INFINITY ? order(x[e]) >> kLow : 0;
            if (o > bound || (o == bound && c <= last_chunk)) {
                const int at = atomicAdd(&sh.n, 1);
                if (at < kCap) sh.key[at] = key_of(x[e], c * N - off + e);
            }
        }
    }
    __syncthreads();
    const int n = sh.n;
    if (n <= kCap) {
        rank_keys(sh, n, k);
        return;
    }
    // ---- too many (a few threads hold most of the large logits): one by one
    uint64_t before = ~0ull;
    for (int r = 0; r < k; ++r) {
        uint64_t v = kNoKey;
        for (int i = tid; i < listed * per; i += kThreads) {
            const int q = i / per, c = c0 + sh.list[q] + (i - q * per) * kThreads;
            if (c >= c1) continue;
            float x[N];
            floats_of<DT>(load_chunk<DT>(row, off, vocab, c), x);
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (x[e] > -INFINITY) {
                    const uint64_t w = key_of(x[e], c * N - off + e);
                    if (w < before && w > v) v = w;
                }
        }
        before = block_max(sh, v);
        if (tid == 0) sh.best[r] = before;
    }
    __syncthreads();
}

template <int DT>
__global__ void __launch_bounds__(kThreads, 4) logprobs_kernel(const __grid_constant__ LpArgs a) {
    constexpr int N = kPer<DT>, UN = 4;   // elements of a chunk, chunks in flight
    __shared__ Shared sh;
    pdl_wait();
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, k = a.top_k;
    const uint32_t row = blockIdx.x / a.segs;
    const int seg = blockIdx.x - row * a.segs;
    const char* base = (const char*)a.logits + (uint64_t)row * a.row_stride * (16 / N);
    const int off = (int)(((uintptr_t)base & 15) / (16 / N));
    const int chunks = (int)(((uint64_t)off + a.vocab + N - 1) / N);
    const int per_seg = (chunks + a.segs - 1) / a.segs;
    const int c0 = seg * per_seg, c1 = min(c0 + per_seg, chunks);
    const float c = a.scale * kLog2e, reach = 64.f / c;

    // ---- the pass: sums against the thread's reference, its maximum and where that is first
    float ref = 0.f, lim = -INFINITY, L = 0.f, E = 0.f, tmax = -INFINITY;
    int tchunk = 0;
    auto take = [&](const uint4& v, int ch) {
        float x[N];
        floats_of<DT>(v, x);
        float cm = x[0];
#pragma unroll
        for (int e = 1; e < N; ++e) cm = fmaxf(cm, x[e]);
        if (cm > tmax) tmax = cm, tchunk = ch;
        if (cm > lim) {
            const float f = lim == -INFINITY ? 0.f : ex2((ref - cm) * c);
            E = lim == -INFINITY ? E : f * fmaf(L, max_nan((ref - cm) * c, -256.f), E);
            L = lim == -INFINITY ? L : f * L;
            ref = cm;
            lim = cm + reach;
        }
        float l2[2] = {0.f, 0.f}, e2[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float d = max_nan((x[e] - ref) * c, -256.f);   // (-inf: weight 0, and not 0 * inf)
            const float w = ex2(d);
            l2[e & 1] += w;
            e2[e & 1] = fmaf(w, d, e2[e & 1]);
        }
        L += l2[0] + l2[1];
        E += e2[0] + e2[1];
    };
    int ch = c0 + tid;
    for (; ch + (UN - 1) * kThreads < c1; ch += UN * kThreads) {
        uint4 v[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) v[u] = load_chunk<DT>(base, off, a.vocab, ch + u * kThreads);
#pragma unroll
        for (int u = 0; u < UN; ++u) take(v[u], ch + u * kThreads);
    }
    for (; ch < c1; ch += kThreads) take(load_chunk<DT>(base, off, a.vocab, ch), ch);

    // ---- the CTA's sums
    float r = lim == -INFINITY ? -INFINITY : ref;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float r2 = __shfl_xor_sync(~0u, r, o), L2 = __shfl_xor_sync(~0u, L, o);
        join(r, L, E, r2, L2, __shfl_xor_sync(~0u, E, o), c);
    }
    if (lane == 0) sh.ref[warp] = r, sh.L[warp] = L, sh.E[warp] = E;
    if (k) select_top<DT>(sh, base, off, a.vocab, c0, c1, tmax, tchunk, k);
    else __syncthreads();
    r = sh.ref[0], L = sh.L[0], E = sh.E[0];
    for (int w = 1; w < kWarps; ++w) join(r, L, E, sh.ref[w], sh.L[w], sh.E[w], c);

    // ---- segments meet in the workspace; the row's last CTA goes on
    if (a.segs > 1) {
        Partial* p = a.partials + (size_t)row * a.segs;
        if (tid < k) __stcg((unsigned long long*)&p[seg].key[tid], sh.best[tid]);
        if (tid == 0) __stcg(reinterpret_cast<float4*>(&p[seg]), make_float4(r, L, E, 0.f));
        __syncthreads();
        if (tid == 0) {
            unsigned was;   // release: the segment's part before its count; acquire: the others'
            asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;"
                         : "=r"(was) : "l"(a.counters + row) : "memory");
            sh.last = was + 1 == (unsigned)a.segs;
            if (sh.last) a.counters[row] = 0;
            sh.n = 0;
        }
        __syncthreads();
        if (!sh.last) return;
        r = -INFINITY, L = E = 0.f;
        if (lane < a.segs) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(&p[lane]));
            r = v.x, L = v.y, E = v.z;
        }
        uint64_t low = kNoKey;   // the best k-th key of a segment: nothing below it counts
        if (k && lane < a.segs) low = __ldcg((const unsigned long long*)&p[lane].key[k - 1]);
#pragma unroll
        for (int o = 16; o; o >>= 1) {   // (in the same order in every warp)
            const float r2 = __shfl_xor_sync(~0u, r, o), L2 = __shfl_xor_sync(~0u, L, o);
            join(r, L, E, r2, L2, __shfl_xor_sync(~0u, E, o), c);
            const uint64_t w = __shfl_xor_sync(~0u, low, o);
            low = w > low ? w : low;
        }
        if (k) {
            for (int i = tid; i < a.segs * k; i += kThreads) {
                const uint64_t v = __ldcg((const unsigned long long*)&p[i / k].key[i % k]);
                if (v != kNoKey && v >= low) sh.key[atomicAdd(&sh.n, 1)] = v;
            }
            __syncthreads();
            rank_keys(sh, sh.n, k);
        }
    }
    // ---- the row's results: lse = scale*r + ln L
    const bool none = r == -INFINITY && L == L;   // no token is possible (and no NaN)
    const float lnL = none ? 0.f : logf(L);
    const float at = r == -INFINITY ? 0.f : r;
    if (tid == 0) {
        if (a.entropy) a.entropy[row] = none ? 0.f : lnL - kLn2 * (E / L);
        if (a.logprob) {
            const int t = a.targets[row];
            a.logprob[row] = (uint32_t)t < a.vocab ? (logit<DT>(base, t) - at) * a.scale - lnL : NAN;
        }
    }
    if (tid < k) {
        const uint64_t v = sh.best[tid];
        const uint64_t o = (uint64_t)row * k + tid;
        a.top_idx[o] = v == kNoKey ? -1 : (int32_t)(0xFFFFFFFFu - (uint32_t)v);
        a.top_lp[o] = v == kNoKey ? (L == L ? -INFINITY : NAN)
                                  : (unorder((uint32_t)(v >> 32)) - at) * a.scale - lnL;
    }
}

int check_logprobs(const GraftLogprobParams* P) {
    clear_error();
    GRAFT_REQUIRE(P, "params pointer is null");
    GRAFT_REQUIRE(P->vocab >= 1 && P->vocab <= 0x7FFFFF00u, "vocab %u out of range", P->vocab);
    GRAFT_REQUIRE(P->rows <= 0x07FFFFFFu, "rows %u out of range", P->rows);
    GRAFT_REQUIRE(P->top_k <= (uint32_t)kMaxTop, "top_k must be at most 32, not %u", P->top_k);
    GRAFT_REQUIRE(P->dtype <= GRAFT_F32, "unknown element type %u", P->dtype);
    GRAFT_REQUIRE(P->row_stride >= P->vocab || P->rows <= 1, "row_stride is below vocab");
    GRAFT_REQUIRE(P->scale >= 0x1p-100f && P->scale <= 0x1p100f,
                  "scale must be positive and finite (2^-100 to 2^100)");
    return GRAFT_OK;
}

// Segments of a row: enough CTAs for several rounds over the SMs, none shorter
// than kMinSeg elements, at most kMaxSegs.
int segments(const GraftLogprobParams* P) {
    const uint64_t rows = P->rows ? P->rows : 1;
    const uint64_t want = (kRounds + rows - 1) / rows;
    const uint64_t most = std::max<uint64_t>(1, P->vocab / kMinSeg);
    return (int)std::min<uint64_t>(std::min<uint64_t>(want, most), kMaxSegs);
}

}  // namespace

extern "C" size_t graft_logprobs_workspace(const GraftLogprobParams* P) {
    if (check_logprobs(P)) return 0;
    const size_t rows = P->rows ? P->rows : 1, segs = segments(P);
    if (segs == 1) return 256;
    return kCounterBytes + rows * segs * sizeof(Partial);
}

extern "C" int graft_logprobs_init(void* ws, size_t ws_bytes, graft_stream_t stream) {
    clear_error();
    GRAFT_REQUIRE(ws && aligned(ws, 256), "the workspace must be 256-byte aligned");
    GRAFT_CUDA(cudaMemsetAsync(ws, 0, ws_bytes, stream));
    return GRAFT_OK;
}

extern "C" int graft_logprobs(const void* logits, const int32_t* targets, float* logprob,
                              float* entropy, float* top_logprob, int32_t* top_index,
                              const GraftLogprobParams* P, void* ws, size_t ws_bytes,
                              graft_stream_t stream) {
    int rc;
    if ((rc = check_logprobs(P))) return rc;
    const size_t need = graft_logprobs_workspace(P);
    GRAFT_REQUIRE(ws && aligned(ws, 256) && ws_bytes >= need,
                  "the workspace must be 256-byte aligned and hold %zu bytes", need);
    if (P->rows == 0) return GRAFT_OK;
    GRAFT_REQUIRE(logits && aligned(logits, P->dtype == GRAFT_F32 ? 4 : 2),
                  "logits must be a buffer aligned to its element type");
    GRAFT_REQUIRE(!logprob == !targets, "targets and logprob go together");
    GRAFT_REQUIRE(P->top_k == 0 || (top_logprob && top_index),
                  "top_logprob and top_index must be given for top_k %u", P->top_k);
    GRAFT_REQUIRE(aligned(targets, 4) && aligned(logprob, 4) && aligned(entropy, 4) &&
                      aligned(top_logprob, 4) && aligned(top_index, 4),
                  "targets and outputs must be 4-byte aligned");
    LpArgs a = {};
    a.logits = logits, a.targets = targets, a.logprob = logprob, a.entropy = entropy;
    a.top_lp = top_logprob, a.top_idx = top_index;
    a.row_stride = P->row_stride, a.rows = P->rows, a.vocab = P->vocab, a.top_k = P->top_k;
    a.scale = P->scale;
    a.segs = segments(P);
    a.counters = (unsigned*)ws;
    a.partials = (Partial*)((char*)ws + kCounterBytes);   // (the counters keep their place in any shape)
    void (*kern)(const LpArgs) = P->dtype == GRAFT_F16    ? logprobs_kernel<GRAFT_F16>
                                 : P->dtype == GRAFT_BF16 ? logprobs_kernel<GRAFT_BF16>
                                                          : logprobs_kernel<GRAFT_F32>;
    return launch_pdl("logprobs", kern, dim3(P->rows * (unsigned)a.segs), kThreads, 0, stream, a);
}
