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
// In a long call of 16-bit logits nothing is at its limit: the pass runs at 4.3 TB/s, about
// 60% of the issue slots and of the MUFU (one exponential an element); four segments a row
// are 2.3 rounds of the CTAs that fit.  fp32 logits are bound by HBM
// (4096 rows of 128256, 5 alternatives: 5.7 TB/s).
//
// The top k come from the threads' own maxima, which the pass finds on the way: each
// thread keeps its largest logit, the round of chunks where that is first, and the
// largest of its other rounds.  A row's last CTA takes every thread's largest over the
// segments; the k-th largest of these bounds the k-th largest logit from below, so only
// rounds that reach it can hold one of the top k.  Those (little more than k) are read
// again, and what reaches the bound is collected and ranked.  Ties go to the lowest
// index: keys are (value, index) pairs, all different.  Segments meet in the workspace,
// and the row's last CTA joins them.
//
// Measured: 777 rows of 128256 in fp16 (199 MB), 5 alternatives: 52.8 us, 3.8 TB/s (46 us
// without alternatives); one row of 201088, 20 alternatives: 9.1 us, without them 4.5;
// 37 rows of 50021 in fp32, 8 alternatives: 9.0 us, without them 5.6.
// Many alternatives of rows that one or two CTAs take (2368 rows or more: one) fall off:
// a thread with two of them in different rounds lists all its chunks, more than kList holds,
// and the row is read once for each alternative.  4096 rows of 128256 in fp32: 5 alternatives
// 372 us, 20 3552, 32 11855; in fp16: 197, 218, 2982.
#include "logits.cuh"

#include <algorithm>
#include <cmath>

using namespace graft;
using namespace graft::dev;

namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kMaxTop = 32, kMaxSegs = 32;
constexpr int kUnroll = 4;           // chunks of a thread's round
constexpr int kCap = 2048;           // keys that are collected at most
constexpr int kList = 1024;          // chunks that are read again at most
constexpr int kMinSeg = 4096;        // elements of a segment, at least
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// CTAs to aim at (777 rows of 128256: 148 x 16 53.5 us, x 10 56.0, x 24 59, x 32 58)
constexpr int kRounds = 148 * 16;
constexpr size_t kCounterBytes = (kRounds * 4 + 255) / 256 * 256;   // a row is cut only if rows < kRounds
constexpr uint64_t kNoKey = 0;       // below every key of a logit that is not -inf

struct Seen {                        // of a thread: besides its largest logit
    int chunk;                       // the first chunk of the first round with it
    uint32_t other;                  // largest of its other rounds, as order()
};
struct Partial {                     // of a segment
    float ref, L, E, pad;
    uint32_t value[kThreads];        // the threads' largest logits as order() (0: none), if k
    Seen seen[kThreads];
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
    union {
        uint64_t key[kCap];
        uint32_t value[kMaxSegs][kThreads];   // the threads' maxima, before keys are collected
    };
    uint64_t best[kMaxTop];
    uint64_t red[kWarps];
    uint32_t most[kThreads];   // the threads' maxima over the segments
    int list[kList];           // chunks
    int n, listed, last;
};
static_assert(kMaxSegs * kThreads * 4 <= kCap * 8, "the maxima fit where the keys go");

__device__ __noinline__ uint64_t block_max(Shared& sh, uint64_t v) {
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

// The k largest of the n different keys sh.key[0..n) into sh.best: a few by
// counting for each key those above it, many one after the other.
__device__ __forceinline__ void rank_keys(Shared& sh, int n, int k) {
    const int tid = threadIdx.x;
    if (n <= kThreads) {
        if (tid < k) sh.best[tid] = kNoKey;
        __syncthreads();
        if (tid < n) {
            const uint64_t v = sh.key[tid];
            int r = 0;
#pragma unroll 4
            for (int j = 0; j < n; ++j) r += sh.key[j] > v;
            if (r < k) sh.best[r] = v;
        }
    } else {
        uint64_t before = ~0ull;
        for (int r = 0; r < k; ++r) {
            uint64_t v = kNoKey;
            for (int i = tid; i < n; i += kThreads) {
                const uint64_t w = sh.key[i];
                if (w < before && w > v) v = w;
            }
            before = block_max(sh, v);
            if (tid == 0) sh.best[r] = before;
        }
    }
    __syncthreads();
}

// A row and its cut.
struct Row {
    const char* base;
    int off;          // elements between a 16-byte boundary and the row
    uint32_t vocab;
    int chunks, per_seg, segs;
};

// A segment's chunks: those wholly in the row are [i0, i1), chunk i0 + t + j*kThreads
// is thread t's j-th; a row's first chunk belongs to thread 0 and its last to
// thread 1 where they lie partly outside (first, last: -1 if not).
struct Span {
    int i0, i1, first, last;
};
template <int N>
__device__ __forceinline__ Span span_of(const Row& w, int seg) {
    const int c0 = min(seg * w.per_seg, w.chunks), c1 = min(c0 + w.per_seg, w.chunks);
    Span sp;
    sp.first = c0 == 0 && c1 > 0 && (w.off || (int)w.vocab < N) ? 0 : -1;
    sp.last = c1 == w.chunks && c1 - 1 > sp.first && c1 > c0 && (w.off + w.vocab) % N ? c1 - 1 : -1;
    sp.i0 = c0 + (sp.first >= 0), sp.i1 = c1 - (sp.last >= 0);
    return sp;
}

__device__ __forceinline__ uint32_t order_or_none(float x) { return x > -INFINITY ? order(x) : 0; }

// The top k keys of a row into sh.best.  own, seen: the thread's largest logit and where it
// is, if the row has one segment; else they stand in `parts`.
template <int DT>
__device__ __forceinline__ void select_top(Shared& sh, const Row& w, const Partial* parts,
                                           uint32_t own, Seen seen, int k) {
    constexpr int N = kPer<DT>;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // ---- each thread's largest over the segments
    if (parts) {
        for (int i = tid; i < w.segs * (kThreads / 4); i += kThreads)
            cp_async16(smem_u32(&sh.value[i / (kThreads / 4)][i % (kThreads / 4) * 4]),
                       &parts[i / (kThreads / 4)].value[i % (kThreads / 4) * 4]);
        cp_async_commit();
        cp_async_wait<0>();
        __syncthreads();
        own = 0;
#pragma unroll 4
        for (int s = 0; s < w.segs; ++s) own = max(own, sh.value[s][tid]);
    }
    sh.most[tid] = own;
    __syncthreads();
    // ---- the k-th largest of these: the bound (1 if there are fewer: whatever is not -inf)
    int above[4] = {0, 0, 0, 0};
#pragma unroll 8
    for (int j = 0; j < kThreads; j += 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(&sh.most[j]);
        above[0] += v.x > own, above[1] += v.y > own, above[2] += v.z > own, above[3] += v.w > own;
    }
    const bool high = above[0] + above[1] + above[2] + above[3] < k;
    const uint32_t low = __reduce_min_sync(~0u, high ? own : 0xFFFFFFFFu);
    if (lane == 0) sh.red[warp] = low;
    if (tid == 0) sh.n = sh.listed = 0;
    __syncthreads();
    uint32_t bound = 0xFFFFFFFFu;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) bound = min(bound, (uint32_t)sh.red[i]);
    bound = max(bound, 1u);

    // ---- the keys of at least `least`, from the rounds that hold such (false: too many)
    auto list = [&](int s, Seen at, uint32_t least) {
        const Span sp = span_of<N>(w, s);
        const bool all = at.other >= least, edge = at.chunk < sp.i0 || at.chunk >= sp.i1;
        const int i0 = all ? sp.i0 + tid : at.chunk;
        const int i1 = all ? sp.i1 : edge ? at.chunk + 1 : min(at.chunk + kUnroll * kThreads, sp.i1);
        const int more = all ? (tid == 0 ? sp.first : tid == 1 ? sp.last : -1) : -1;
        const int count = (max(i1 - i0, 0) + kThreads - 1) / kThreads + (more >= 0);
        int to = atomicAdd(&sh.listed, count);
        if (to + count > kList) return;
        for (int c = i0; c < i1; c += kThreads) sh.list[to++] = c;
        if (more >= 0) sh.list[to] = more;
    };
    auto collect = [&](int c, uint32_t least, uint32_t most) {
        float x[N];
        floats_of<DT>(load_chunk<DT>(w.base, w.off, w.vocab, c), x);
        uint32_t hits = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const uint32_t o = order_or_none(x[e]);
            hits |= (uint32_t)(o >= least && o <= most) << e;
        }
        if (!hits) return;
        int to = atomicAdd(&sh.n, __popc(hits));
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (hits >> e & 1) {
                if (to < kCap) sh.key[to] = key_of(x[e], c * N - w.off + e);
                ++to;
            }
    };
    bool done = false;
    uint32_t least = bound;
#pragma unroll 1
    for (int pass = 0; pass < 2 && !done; ++pass, ++least) {
        // (many equal to the bound, in a row of which all but a few tokens have one lowest
        // value, say, are passed over by the second pass: those above it)
        if (pass) {
            __syncthreads();
            if (tid == 0) sh.n = sh.listed = 0;
            __syncthreads();
        }
        if (own >= least) {
            uint32_t segs = 1;
            if (parts) {
                segs = 0;
                if (pass == 0) {
#pragma unroll 4
                    for (int s = 0; s < w.segs; ++s) segs |= (uint32_t)(sh.value[s][tid] >= least) << s;
                } else {   // (keys lie there now)
#pragma unroll 4
                    for (int s = 0; s < w.segs; ++s)
                        segs |= (uint32_t)(__ldcg(&parts[s].value[tid]) >= least) << s;
                }
            }
            for (; segs; segs &= segs - 1) {
                const int s = __ffs(segs) - 1;
                if (parts) {
                    const uint2 v = __ldcg(reinterpret_cast<const uint2*>(&parts[s].seen[tid]));
                    seen = Seen{(int)v.x, v.y};
                }
                list(s, seen, least);
            }
        }
        __syncthreads();
        if (sh.listed > kList) continue;
        for (int i = tid; i < sh.listed; i += kThreads) collect(sh.list[i], least, ~0u);
        __syncthreads();
        // (room for the equal ones: fewer than k, and one more round of the CTA's chunks)
        done = sh.n <= (pass ? kCap - kThreads * N - kMaxTop : kCap);
    }
    if (done && least > bound + 1) {   // .. and the first of the equal ones in their order
        const int want = sh.n + k;
        for (int c = 0; c < w.chunks && sh.n < want; c += kThreads) {
            __syncthreads();   // (sh.n has been read)
            if (c + tid < w.chunks) collect(c + tid, bound, bound);
            __syncthreads();
        }
    }
    __syncthreads();
    if (done) {
        rank_keys(sh, sh.n, k);
        return;
    }
    // ---- a few threads hold most of the large logits: one by one
    uint64_t before = ~0ull;
    for (int r = 0; r < k; ++r) {
        uint64_t v = kNoKey;
        for (int c = tid; c < w.chunks; c += kThreads) {
            float x[N];
            floats_of<DT>(load_chunk<DT>(w.base, w.off, w.vocab, c), x);
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (x[e] > -INFINITY) {
                    const uint64_t y = key_of(x[e], c * N - w.off + e);
                    if (y < before && y > v) v = y;
                }
        }
        before = block_max(sh, v);
        if (tid == 0) sh.best[r] = before;
    }
    __syncthreads();
}

// (nine CTAs an SM, 56 registers: 52.3 us for 777 rows of 128256; ten 53.3)
template <int DT>
__global__ void __launch_bounds__(kThreads, 9) logprobs_kernel(const __grid_constant__ LpArgs a) {
    constexpr int N = kPer<DT>, UN = kUnroll;
    __shared__ Shared sh;
    pdl_wait();
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, k = a.top_k;
    const uint32_t row = blockIdx.x / a.segs;
    const int seg = blockIdx.x - row * a.segs;
    const char* base = (const char*)a.logits + (uint64_t)row * a.row_stride * (16 / N);
    const int off = (int)(((uintptr_t)base & 15) / (16 / N));
    const int chunks = (int)(((uint64_t)off + a.vocab + N - 1) / N);
    const Row w{base, off, a.vocab, chunks, (chunks + a.segs - 1) / a.segs, a.segs};
    const Span sp = span_of<N>(w, seg);
    const float c = a.scale * kLog2e, reach = 64.f / c;

    // ---- the pass: sums against the thread's reference, its maximum and where that is first
    float ref = 0.f, lim = -INFINITY, tmax = -INFINITY, other = -INFINITY;
    float L2[2] = {0.f, 0.f}, E2[2] = {0.f, 0.f};   // two partial sums each
    int round = 0;
    auto take = [&](const uint4 (&v)[UN], int ch) {   // chunks ch, ch + kThreads, ..
        float gm;
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const float m = chunk_max<DT>(v[u]);
            gm = u ? fmaxf(gm, m) : m;
        }
        other = fmaxf(other, fminf(gm, tmax));
        round = gm > tmax ? ch : round;
        tmax = fmaxf(tmax, gm);
        if (gm > lim) {
            if (lim > -INFINITY) {
                const float a = (ref - gm) * c, f = ex2(a), b = max_nan(a, -256.f);
#pragma unroll
                for (int i = 0; i < 2; ++i) E2[i] = f * fmaf(L2[i], b, E2[i]), L2[i] *= f;
            }
            ref = gm;
            lim = __fadd_rd(gm, reach);   // (rounded up, it might let 2^128 through)
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const uint32_t w4[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                float d0, d1;
                if constexpr (DT == GRAFT_F32) {
                    d0 = __uint_as_float(w4[e]) - ref, d1 = __uint_as_float(w4[e + 1]) - ref;
                } else {
                    minus<DT>(w4[e / 2], ref, d0, d1);
                }
                // (a weight of -inf is 0, and must not be 0 * inf)
                d0 = max_nan(d0 * c, -256.f), d1 = max_nan(d1 * c, -256.f);
                const float w0 = ex2(d0), w1 = ex2(d1);
                L2[0] += w0, L2[1] += w1;
                E2[0] = fmaf(w0, d0, E2[0]), E2[1] = fmaf(w1, d1, E2[1]);
            }
        }
    };
    int ch = sp.i0 + tid;
    const char* from = base + ((int64_t)ch * N - off) * (16 / N);
#pragma unroll 1
    for (; ch + (UN - 1) * kThreads < sp.i1; ch += UN * kThreads, from += UN * kThreads * 16) {
        uint4 v[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) v[u] = ld_stream(from + u * kThreads * 16);
        take(v, ch);
    }
    // what is left, and the row's edge, as rounds with empty chunks
    const int edge = tid == 0 ? sp.first : tid == 1 ? sp.last : -1;
#pragma unroll 1
    for (int part = 0; part < 2; ++part) {
        if (part ? edge < 0 : ch >= sp.i1) continue;
        constexpr uint32_t none = DT == GRAFT_F32 ? 0xFF800000u : DT == GRAFT_F16 ? 0xFC00FC00u : 0xFF80FF80u;
        uint4 v[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            v[u] = make_uint4(none, none, none, none);
            if (part) {
                if (u == 0) v[u] = load_chunk<DT>(base, off, a.vocab, edge);
            } else if (ch + u * kThreads < sp.i1) {
                v[u] = ld_stream(from + u * kThreads * 16);
            }
        }
        take(v, part ? edge : ch);
    }

    // ---- the CTA's sums: against the warp's largest reference, then the warps'
    float L, E, r = lim == -INFINITY ? -INFINITY : ref;
    {
        L = L2[0] + L2[1], E = E2[0] + E2[1];
        float m = r;
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        const float b = r == -INFINITY ? 0.f : (r - m) * c, f = r == -INFINITY ? 0.f : ex2(b);
        E = f * fmaf(L, max_nan(b, -256.f), E);
        L *= f;
        r = m;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            L += __shfl_xor_sync(~0u, L, o);
            E += __shfl_xor_sync(~0u, E, o);
        }
    }
    if (lane == 0) sh.ref[warp] = r, sh.L[warp] = L, sh.E[warp] = E;
    __syncthreads();
    if (warp == 0) {   // (the others' stay their own: the first warp writes the results)
        r = -INFINITY, L = E = 0.f;
        if (lane < kWarps) r = sh.ref[lane], L = sh.L[lane], E = sh.E[lane];
#pragma unroll
        for (int o = kWarps / 2; o; o >>= 1) {
            const float r2 = __shfl_xor_sync(~0u, r, o), m2 = __shfl_xor_sync(~0u, L, o);
            join(r, L, E, r2, m2, __shfl_xor_sync(~0u, E, o), c);
        }
    }

    const uint32_t mine = order_or_none(tmax);
    const Seen seen{round, order_or_none(other)};
    // ---- segments meet in the workspace; the row's last CTA goes on
    if (a.segs > 1) {
        Partial* p = a.partials + (size_t)row * a.segs;
        if (k) {
            __stcg(&p[seg].value[tid], mine);
            __stcg(reinterpret_cast<uint2*>(&p[seg].seen[tid]), make_uint2(seen.chunk, seen.other));
        }
        if (tid == 0) __stcg(reinterpret_cast<float4*>(&p[seg]), make_float4(r, L, E, 0.f));
        __syncthreads();
        if (tid == 0) {
            unsigned was;   // release: the segment's part before its count; acquire: the others'
            asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;"
                         : "=r"(was) : "l"(a.counters + row) : "memory");
            sh.last = was + 1 == (unsigned)a.segs;
            if (sh.last) a.counters[row] = 0;
        }
        __syncthreads();
        if (!sh.last) return;
        r = -INFINITY, L = E = 0.f;
        if (lane < a.segs) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(&p[lane]));
            r = v.x, L = v.y, E = v.z;
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const float r2 = __shfl_xor_sync(~0u, r, o), L2 = __shfl_xor_sync(~0u, L, o);
            join(r, L, E, r2, L2, __shfl_xor_sync(~0u, E, o), c);
        }
    }
    if (k) select_top<DT>(sh, w, a.segs > 1 ? a.partials + (size_t)row * a.segs : nullptr,
                          mine, seen, k);
    // ---- the row's results, by the first warp: lse = scale*r + ln L
    if (warp) return;
    r = __shfl_sync(~0u, r, 0), L = __shfl_sync(~0u, L, 0), E = __shfl_sync(~0u, E, 0);
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
