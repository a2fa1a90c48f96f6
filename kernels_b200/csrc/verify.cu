// verify.cu -- trees of drafted tokens: their masks and positions, and which of the
// drafted tokens stand against the target's probabilities.
//
//   p = softmax(scale z), q = softmax(draft_scale z'), r = p, R = 1
//   child c accepted:  u_c q(x_c) R < r(x_c);   else  r <- max(r - R q, 0), R <- sum r
//   next = smallest v with r(v) > 0 and  sum_{w <= v} r(w) > u R
//
// Two kernels.  The first reads the rows of tokens that have children (a leaf's row matters
// only if it turns out to be the last) and leaves each segment's (reference, sum).  The
// second gives a sequence a cluster of CTAs: whether a token's first child is accepted
// follows from two logits and two sums, for all tokens at once, so the walk down the tree is
// a few steps in shared memory; then the cluster goes over the last token's row (and the
// draft's, where a child was rejected) in fp64: cumulative sums decide about `next`, and at 10^5
// tokens an error of 2^-24 would move one draw in a hundred to a neighbour.
#include "kv_common.cuh"

#include <algorithm>
#include <cmath>

using namespace graft;
using namespace graft::dev;

namespace {

// ------------------------------------------------------------ masks of a tree --
struct TreeArgs {
    const int32_t *parents, *start, *cu;
    uint32_t n_seqs, max_tokens, max_len, tokens, window, words;
    uint32_t* mask;
    uint64_t mask_stride;
    int32_t* positions;
};

__device__ unsigned g_tree_err;

constexpr int kTreeThreads = 128;

// A CTA a sequence, a thread a token: up its ancestors, one word of the mask at a time.
__global__ void __launch_bounds__(kTreeThreads) draft_tree_kernel(const __grid_constant__ TreeArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const int b = blockIdx.x;
    const int c0 = a.cu[b], n = a.cu[b + 1] - c0, start = a.start[b];
    if (c0 < 0 || n < 0 || n > (int)a.max_tokens || (uint64_t)c0 + (uint64_t)n > a.tokens || start < 0 ||
        (uint64_t)((int64_t)start + n) > a.max_len) {
        if (threadIdx.x == 0) atomicOr(&g_tree_err, (unsigned)GRAFT_KV_EBOUNDS);
        return;
    }
    for (int i = threadIdx.x; i < n; i += kTreeThreads) {
        uint32_t* row = a.mask + (uint64_t)(c0 + i) * a.mask_stride;
        int at = (int)a.words - 1, depth = 0, j = i;
        uint32_t word = 0;
        for (;;) {
            if (a.window == 0 || depth < (int)a.window) {
                for (; at > j >> 5; --at) row[at] = word, word = 0;
                word |= 1u << (j & 31);
            }
            const int p = j ? a.parents[c0 + j] : -1;
            if (p < 0 || p >= j) break;
            j = p, ++depth;
        }
        for (; at >= 0; --at) row[at] = word, word = 0;
        if (a.positions) a.positions[c0 + i] = start + depth;
    }
}

// ------------------------------------------------------------------ verifying --
constexpr int kMaxTree = 1024;       // tokens of a sequence
constexpr int kRowThreads = 128, kRowWarps = kRowThreads / 32;
constexpr int kMaxSegs = 32, kMinSeg = 4096;
constexpr int kRounds = 148 * 16;    // CTAs to aim at
constexpr int kWalkThreads = 512, kWalkWarps = kWalkThreads / 32, kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;

struct VerifyArgs {
    const void *logits, *draft;
    const int32_t *tokens, *parents, *cu;
    const float *uniform, *uniform_next;
    int32_t *count, *path, *next;
    uint64_t row_stride, draft_stride;
    uint32_t n_seqs, rows, max_tokens, vocab;
    float scale, draft_scale;
    int segs;
    uint64_t* parts;   // [draft: 2][rows][segs]: (reference, sum), or greedy the largest key
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// fp32 in the order of unsigned integers, NaN above all (-0 = +0)
__device__ __forceinline__ uint32_t order(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return x == x ? b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u) : 0xFFFFFFFFu;
}
constexpr uint32_t kOrderInf = 0xFF800000u, kOrderNone = 0x007FFFFFu;   // of +inf and -inf
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) {
    return ((uint64_t)order(x) << 32) | (0xFFFFFFFFu - index);
}
__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }

template <int DT>
__device__ __forceinline__ float logit(const void* row, uint32_t i) {
    if constexpr (DT == GRAFT_F32) return ((const float*)row)[i];
    const uint16_t w = ((const uint16_t*)row)[i];
    return DT == GRAFT_F16 ? h2f(w) : bf2f(w);
}
template <int DT>
constexpr int kSize = DT == GRAFT_F32 ? 4 : 2;

// Elements v .. v + 7 of a row; those from vocab on are -inf and are not read.
template <int DT>
__device__ __forceinline__ void load8(const void* row, uint32_t v, uint32_t vocab, float (&x)[8]) {
    const char* p = (const char*)row + (uint64_t)v * kSize<DT>;
    if (v + 8 <= vocab && ((uintptr_t)p & 15) == 0) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        if constexpr (DT == GRAFT_F32) {
            const uint4 b = *reinterpret_cast<const uint4*>(p + 16);
            x[0] = __uint_as_float(a.x), x[1] = __uint_as_float(a.y), x[2] = __uint_as_float(a.z);
            x[3] = __uint_as_float(a.w), x[4] = __uint_as_float(b.x), x[5] = __uint_as_float(b.y);
            x[6] = __uint_as_float(b.z), x[7] = __uint_as_float(b.w);
        } else {
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = unpack2<DT>(w[i]);
                x[2 * i] = f.x, x[2 * i + 1] = f.y;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = v + i < vocab ? logit<DT>(row, v + i) : -INFINITY;
    }
}

// Whether row r is a token that has children (every thread of the CTA asks).
__device__ __forceinline__ bool has_children(const VerifyArgs& a, int r) {
    __shared__ int sh[2];
    for (uint32_t s0 = 0;; s0 += blockDim.x) {
        const uint32_t s = s0 + threadIdx.x;
        bool here = false;
        if (s < a.n_seqs) {
            const int c = a.cu[s], e = a.cu[s + 1];
            here = c <= r && r < e;
            if (here) sh[0] = c, sh[1] = e;
        }
        const int found = __syncthreads_count(here);
        if (found == 1) break;
        if (found > 1 || s0 + blockDim.x >= a.n_seqs) return false;
    }
    const int c0 = sh[0], n = sh[1] - c0, i = r - c0;
    if (c0 < 0 || n > (int)a.max_tokens || (uint64_t)c0 + (uint64_t)n > a.rows) return false;
    if (!a.parents) return i + 1 < n;
    bool mine = false;
    for (int j = i + 1 + threadIdx.x; j < n; j += blockDim.x) mine |= a.parents[c0 + j] == i;
    return __syncthreads_or(mine);
}

// A segment of a row: its largest logit and sum of exp(scale (z - it)), or the largest key.
template <int DT, bool GREEDY>
__global__ void __launch_bounds__(kRowThreads) verify_rows_kernel(const __grid_constant__ VerifyArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ float2 sh[kRowWarps];
    __shared__ uint64_t sh_key[kRowWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t row = blockIdx.x / a.segs, seg = blockIdx.x - row * a.segs;
    if (!has_children(a, row)) return;
    const bool of_draft = blockIdx.y;
    const char* base = of_draft ? (const char*)a.draft + row * a.draft_stride * kSize<DT>
                                : (const char*)a.logits + row * a.row_stride * kSize<DT>;
    const float c = (of_draft ? a.draft_scale : a.scale) * kLog2e;
    const uint32_t per = ((a.vocab + a.segs - 1) / a.segs + 7) / 8 * 8;
    const uint32_t v0 = seg * per, v1 = min(a.vocab, v0 + per);
    float m = -INFINITY, L = 0.f;
    uint64_t key = 0;
    for (uint32_t v = v0 + tid * 8; v < v1; v += kRowThreads * 8) {
        float x[8];
        load8<DT>(base, v, v1, x);
        if constexpr (GREEDY) {
#pragma unroll
            for (int i = 0; i < 8; ++i) key = max64(key, v + i < v1 ? key_of(x[i], v + i) : 0);
        } else {
            float mx = x[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) mx = fmaxf(mx, x[i]);
            if (mx > m) {
                L *= m == -INFINITY ? 0.f : ex2((m - mx) * c);
                m = mx;
            }
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int i = 0; i < 8; ++i) L += ex2((x[i] - ref) * c);
        }
    }
    uint64_t* out = a.parts + ((uint64_t)of_draft * a.rows + row) * a.segs + seg;
    if constexpr (GREEDY) {
#pragma unroll
        for (int o = 16; o; o >>= 1) key = max64(key, __shfl_xor_sync(~0u, key, o));
        if (lane == 0) sh_key[warp] = key;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < kRowWarps; ++w) key = max64(key, sh_key[w]);
            *out = key;
        }
    } else {
        auto join = [&](float m2, float L2) {
            const float top = fmaxf(m, m2), ref = top == -INFINITY ? 0.f : top;
            L = (m == -INFINITY ? L : L * ex2((m - ref) * c)) + (m2 == -INFINITY ? L2 : L2 * ex2((m2 - ref) * c));
            m = top;
        };
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const float m2 = __shfl_xor_sync(~0u, m, o);
            join(m2, __shfl_xor_sync(~0u, L, o));
        }
        if (lane == 0) sh[warp] = make_float2(m, L);
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < kRowWarps; ++w) join(sh[w].x, sh[w].y);
            *reinterpret_cast<float2*>(out) = make_float2(m, L);
        }
    }
}

// ---- the walk: a cluster a sequence
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// Stores 64 bits at the same place of another CTA of the cluster.
__device__ __forceinline__ void store_remote(const void* at, uint32_t rank, uint64_t v) {
    asm volatile("{\n\t.reg .b32 to;\n\tmapa.shared::cluster.u32 to, %0, %1;\n\t"
                 "st.shared::cluster.b64 [to], %2;\n\t}" ::"r"(smem_u32(at)), "r"(rank), "l"(v)
                 : "memory");
}

enum Flag : uint8_t { kRejected, kAccepted, kAsk, kIgnored };   // kAsk: the whole row decides

struct Walk {
    int first[kMaxTree];            // child, or kMaxTree
    int token[kMaxTree];
    float2 stat[kMaxTree], stat_q[kMaxTree];
    double chance[kMaxTree];        // r of a token under its parent, before any rejection
    double mass[kMaxTree];          // R after so many rejections of the current token's children
    int16_t parent[kMaxTree], sibling[kMaxTree];   // sibling: the next one, or -1
    uint8_t flag[kMaxTree];
    bool again[kMaxTree];           // an earlier sibling has the same token
    uint64_t part[2][kMaxCluster * kWalkWarps];
};

template <int DT, bool GREEDY>
__global__ void __launch_bounds__(kWalkThreads) verify_walk_kernel(const __grid_constant__ VerifyArgs a, int ctas) {
    extern __shared__ __align__(16) uint8_t smem[];
    Walk& sh = *reinterpret_cast<Walk*>(smem);
    pdl_wait();
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = cluster_rank(), b = blockIdx.x / ctas, NW = ctas * kWalkWarps;
    const int c0 = a.cu[b], n = a.cu[b + 1] - c0;
    if (c0 < 0 || n <= 0 || n > (int)a.max_tokens || (uint64_t)c0 + (uint64_t)n > a.rows) {
        if (rank == 0 && tid == 0) a.count[b] = 0, a.next[b] = -1;
        return;   // (the whole cluster)
    }
    const bool drawn = !GREEDY && a.draft;
    const double scale = a.scale, scale_q = a.draft_scale;
    auto row_of = [&](int i) { return (const char*)a.logits + (uint64_t)(c0 + i) * a.row_stride * kSize<DT>; };
    auto draft_of = [&](int i) { return (const char*)a.draft + (uint64_t)(c0 + i) * a.draft_stride * kSize<DT>; };
    auto usable = [](float2 s) { return s.x < INFINITY && s.y > 0.f && s.y < INFINITY; };

    // ---- the tree
    for (int i = tid; i < n; i += kWalkThreads) {
        const int p = i == 0 ? -1 : a.parents ? a.parents[c0 + i] : i - 1;
        sh.parent[i] = p >= 0 && p < i ? p : -1;
        sh.token[i] = a.tokens[c0 + i];
        sh.first[i] = kMaxTree;
    }
    __syncthreads();
    for (int i = 1 + tid; i < n; i += kWalkThreads) {
        const int p = sh.parent[i];
        if (p >= 0) atomicMin(&sh.first[p], i);
        int s = -1;
        if (a.parents && p >= 0)
            for (int j = i + 1; j < n; ++j)
                if (sh.parent[j] == p) {
                    s = j;
                    break;
                }
        sh.sibling[i] = s;
    }
    __syncthreads();
    // ---- sums of the rows of tokens with children, a warp a row
    for (int i = warp; i < n; i += kWalkWarps)
        if (sh.first[i] < kMaxTree) {
            for (int which = 0; which < (drawn ? 2 : 1); ++which) {
                const uint64_t* parts = a.parts + ((uint64_t)which * a.rows + c0 + i) * a.segs;
                uint64_t v = lane < a.segs ? parts[lane] : 0;
                if constexpr (GREEDY) {
#pragma unroll
                    for (int o = 16; o; o >>= 1) v = max64(v, __shfl_xor_sync(~0u, v, o));
                    if (lane == 0) {
                        const uint32_t top = v >> 32;
                        const bool ok = top > kOrderNone && top < kOrderInf;
                        sh.stat[i] = make_float2(__int_as_float(ok ? (int)(0xFFFFFFFFu - (uint32_t)v) : -1), 0.f);
                    }
                } else {
                    const float c = (which ? a.draft_scale : a.scale) * kLog2e;
                    float m = lane < a.segs ? __uint_as_float((uint32_t)v) : -INFINITY;
                    float L = lane < a.segs ? __uint_as_float((uint32_t)(v >> 32)) : 0.f;
                    float top = m;
#pragma unroll
                    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
                    L = m == -INFINITY ? L : L * ex2((m - top) * c);
#pragma unroll
                    for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(~0u, L, o);
                    if (lane == 0) (which ? sh.stat_q : sh.stat)[i] = make_float2(top, L);
                }
            }
        }
    __syncthreads();
    // ---- what each child's own chances say
    for (int i = 1 + tid; i < n; i += kWalkThreads) {
        const int p = sh.parent[i], x = sh.token[i];
        uint8_t f = kIgnored;
        bool again = false;
        double chance = 0;
        if (p >= 0 && (uint32_t)x < a.vocab) {
            if constexpr (GREEDY) {
                f = __float_as_int(sh.stat[p].x) == x ? kAccepted : kRejected;
            } else if (usable(sh.stat[p])) {
                for (int e = sh.first[p]; e != i; e = sh.sibling[e]) again |= sh.token[e] == x;
                chance = exp(((double)logit<DT>(row_of(p), x) - sh.stat[p].x) * scale) / sh.stat[p].y;
                if (!drawn) {
                    f = kRejected;   // (decided below)
                } else if (usable(sh.stat_q[p])) {
                    const double q = exp(((double)logit<DT>(draft_of(p), x) - sh.stat_q[p].x) * scale_q) / sh.stat_q[p].y;
                    f = sh.first[p] != i ? kAsk : (double)a.uniform[c0 + i] * q < chance ? kAccepted : kRejected;
                }
            }
        }
        sh.flag[i] = f, sh.again[i] = again, sh.chance[i] = chance;
    }
    __syncthreads();
    if constexpr (!GREEDY) {
        if (!drawn) {
            // r is p without the earlier siblings' tokens
            for (int i = 1 + tid; i < n; i += kWalkThreads)
                if (sh.flag[i] == kRejected && !sh.again[i]) {
                    double R = 1;
                    for (int e = sh.first[sh.parent[i]]; e != i; e = sh.sibling[e])
                        if (sh.flag[e] != kIgnored && !sh.again[e]) R -= sh.chance[e];
                    // (where little is left of 1, the sums' own errors count: the row decides)
                    sh.mass[i] = R;
                }
            __syncthreads();
            for (int i = 1 + tid; i < n; i += kWalkThreads)
                if (sh.flag[i] == kRejected && !sh.again[i]) {
                    const double R = sh.mass[i];
                    sh.flag[i] = R < 0x1p-10 ? kAsk : (double)a.uniform[c0 + i] * R < sh.chance[i] ? kAccepted : kRejected;
                }
            __syncthreads();
        }
    }

    // ---- passes of the cluster over a row: each warp a piece of whole steps of 256 tokens
    const uint32_t piece = ((a.vocab + NW - 1) / NW + 255) / 256 * 256;
    const uint64_t lo64 = (uint64_t)(rank * kWalkWarps + warp) * piece;
    const uint32_t lo = (uint32_t)min(lo64, (uint64_t)a.vocab), hi = (uint32_t)min(lo64 + piece, (uint64_t)a.vocab);
    int turn = 0;
    // every warp's value, at every CTA
    auto spread = [&](uint64_t v) -> const uint64_t* {
        uint64_t* to = sh.part[turn];
        turn ^= 1;
        if (lane < ctas) store_remote(to + rank * kWalkWarps + warp, lane, v);
        cluster_sync();
        return to;
    };
    auto warp_sum64 = [&](double x) {
#pragma unroll
        for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
        return x;
    };
    auto total = [&](const uint64_t* parts) {   // (the same order of sums in every thread)
        double s = 0;
        for (int w = lane; w < NW; w += 32) s += __longlong_as_double(parts[w]);
        return warp_sum64(s);
    };

    // The last token's row: references, sums, rejections.
    int cur = 0, cnt = 1;
    float ref = 0.f, ref_q = 0.f;
    double Lp = 0, Lq = 0;
    int m = 0, from = 0;       // rejections that count; those before `from` left nothing
    bool summed = false;       // Lp and Lq are those of cur
    // r of token v with target and draft exponentials ep and eq, after k rejections
    auto left = [&](double ep, double eq, int k) {
        double r = ep / Lp;
        const double q = eq / Lq;
        for (int i = from; i < k; ++i) r = fmax(r - sh.mass[i] * q, 0.0);
        return r;
    };
    auto gone = [&](uint32_t v, int stop) {   // not drawn: the token of a rejected child before `stop`
        for (int e = sh.first[cur]; e >= 0 && e < kMaxTree && e != stop; e = sh.sibling[e])
            if (sh.flag[e] == kRejected && !sh.again[e] && sh.token[e] == (int)v) return true;
        return false;
    };
    // Sum over the warp's piece of what f makes of eight tokens of the row (and of the draft's).
    auto sweep = [&](bool both, auto f) {
        const void *zp = row_of(cur), *zq = both ? draft_of(cur) : nullptr;
        double s = 0;
        for (uint32_t v = lo + lane * 8; v < hi; v += 256) {
            float x[8], y[8];
            load8<DT>(zp, v, a.vocab, x);
            if (both) load8<DT>(zq, v, a.vocab, y);
            s += f(x, y, v);
        }
        return s;
    };
    auto expo = [&](float x, float r, double sc) { return exp(((double)x - r) * sc); };
    auto sums = [&]() {        // Lp (and Lq) in 64 bits
        if (summed) return;
        double sq = 0;
        const double sp = sweep(true, [&](const float (&x)[8], const float (&y)[8], uint32_t) {
            double s = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) s += expo(x[i], ref, scale), sq += expo(y[i], ref_q, scale_q);
            return s;
        });
        const uint64_t* p = spread(__double_as_longlong(warp_sum64(sp)));
        Lp = total(p);
        p = spread(__double_as_longlong(warp_sum64(sq)));
        Lq = total(p);
        summed = true;
    };
    auto mass_of = [&](int k) {   // the warps' sums of r after k rejections
        const double s = sweep(true, [&](const float (&x)[8], const float (&y)[8], uint32_t) {
            double t = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) t += left(expo(x[i], ref, scale), expo(y[i], ref_q, scale_q), k);
            return t;
        });
        return spread(__double_as_longlong(warp_sum64(s)));
    };
    auto set_mass = [&](int k, double R) {   // (every thread has the same R)
        __syncthreads();
        if (tid == 0) sh.mass[k] = R;
        __syncthreads();
    };
    auto without = [&](int stop) {   // the warps' sums of p's exponentials without rejected tokens
        const double s = sweep(false, [&](const float (&x)[8], const float (&)[8], uint32_t v) {
            double t = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) t += m && gone(v + i, stop) ? 0.0 : expo(x[i], ref, scale);
            return t;
        });
        return spread(__double_as_longlong(warp_sum64(s)));
    };

    if (rank == 0)
        for (int i = tid; i < n; i += kWalkThreads) a.path[c0 + i] = i ? -1 : c0;
    __syncthreads();
    for (;;) {   // (every thread of the cluster takes the same way)
        int c = sh.first[cur];
        m = from = 0, summed = false;
        ref = sh.stat[cur].x, ref_q = sh.stat_q[cur].x;
        if (drawn) set_mass(0, 1.0);
        int took = -1;
        if (c < kMaxTree)
            for (; c >= 0; c = sh.sibling[c]) {
                uint8_t f = sh.flag[c];
                if (f == kIgnored) continue;
                if (f == kAsk) {
                    const double u = a.uniform[c0 + c];
                    const uint32_t x = sh.token[c];
                    if (drawn) {
                        sums();
                        const double ep = expo(logit<DT>(row_of(cur), x), ref, scale);
                        const double eq = expo(logit<DT>(draft_of(cur), x), ref_q, scale_q);
                        f = u * (eq / Lq) * sh.mass[m] < left(ep, eq, m) ? kAccepted : kRejected;
                    } else {
                        double R = total(without(c));
                        const double e = expo(logit<DT>(row_of(cur), x), ref, scale);
                        f = u * R < e ? kAccepted : kRejected;
                        __syncthreads();
                        if (tid == 0) sh.flag[c] = f;
                        __syncthreads();
                    }
                }
                if (f == kAccepted) {
                    took = c;
                    break;
                }
                ++m;
                if (drawn) {
                    // R is needed for the next child and for the draw; the last one's is found there
                    if (sh.sibling[c] >= 0) {
                        sums();
                        double R = total(mass_of(m));
                        if (!(R > 0)) from = m, R = 1;
                        set_mass(m, R);
                    }
                }
            }
        if (took < 0) break;
        cur = took;
        if (rank == 0 && tid == 0) a.path[c0 + cnt] = c0 + cur;
        ++cnt;
        __syncthreads();   // (before masses and flags of the next token's children)
    }
    if (rank == 0 && tid == 0) a.count[b] = cnt;

    // ---- next
    const bool inner = sh.first[cur] < kMaxTree;
    if constexpr (GREEDY) {
        int best = __float_as_int(sh.stat[cur].x);
        if (!inner) {
            uint64_t key = 0;
            for (uint32_t v = lo + lane * 8; v < hi; v += 256) {
                float x[8];
                load8<DT>(row_of(cur), v, a.vocab, x);
#pragma unroll
                for (int i = 0; i < 8; ++i) key = max64(key, v + i < a.vocab ? key_of(x[i], v + i) : 0);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) key = max64(key, __shfl_xor_sync(~0u, key, o));
            const uint64_t* p = spread(key);
            key = 0;
            for (int w = 0; w < NW; ++w) key = max64(key, p[w]);
            const uint32_t top = key >> 32;
            best = top > kOrderNone && top < kOrderInf ? (int)(0xFFFFFFFFu - (uint32_t)key) : -1;
        }
        if (rank == 0 && tid == 0) a.next[b] = best;
    } else {
        if (!inner) {   // a leaf's row has not been read yet
            float top = -INFINITY;
            for (uint32_t v = lo + lane * 8; v < hi; v += 256) {
                float x[8];
                load8<DT>(row_of(cur), v, a.vocab, x);
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, x[i]);   // (a NaN shows in the sum)
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
            const uint64_t* p = spread(order(top));
            uint64_t most = 0;
            for (int w = 0; w < NW; ++w) most = max64(most, p[w]);
            const uint32_t o = (uint32_t)most;
            ref = __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xFFFFFFFFu));
        }
        const uint64_t* parts = nullptr;
        double R = 0;
        int k = drawn ? m : 0;
        if (ref > -INFINITY && ref < INFINITY) {
            if (k) {
                sums();
                parts = mass_of(k);
                R = total(parts);
                if (!(R > 0)) k = 0;   // nothing is left: p again
            }
            if (!k) {
                parts = without(-1);
                R = total(parts);
                if (!(R > 0) && m) {
                    m = 0;
                    parts = without(-1);
                    R = total(parts);
                }
            }
        }
        if (!(R > 0 && R < INFINITY)) {
            if (rank == 0 && tid == 0) a.next[b] = -1;
        } else {
            // ---- the warp whose piece the sum passes u R in, then the token
            const double goal = (double)a.uniform_next[b] * R;
            int owner = -1, last = 0;
            double before = 0, base = 0;
            for (int w = 0; w < NW; ++w) {
                const double s = __longlong_as_double(parts[w]);
                if (s > 0) last = w;
                if (owner < 0 && s > 0 && before + s > goal) owner = w, base = before;
                before += s;
            }
            const bool found = owner >= 0;
            if (!found) owner = last;
            if (owner == rank * kWalkWarps + warp) {
                const void *zp = row_of(cur), *zq = k ? draft_of(cur) : nullptr;
                int best = -1, final_one = -1;
                for (uint32_t v0 = lo; v0 < hi && best < 0; v0 += 256) {
                    const uint32_t v = v0 + lane * 8;
                    double r[8], s = 0;
                    float x[8], y[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) r[i] = 0;
                    if (v < hi) {
                        load8<DT>(zp, v, a.vocab, x);
                        if (k) load8<DT>(zq, v, a.vocab, y);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const double ep = expo(x[i], ref, scale);
                            r[i] = k ? left(ep, expo(y[i], ref_q, scale_q), k) : m && gone(v + i, -1) ? 0.0 : ep;
                            s += r[i];
                        }
                    }
                    double upto = s;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const double t = __shfl_up_sync(~0u, upto, o);
                        if (lane >= o) upto += t;
                    }
                    int mine = -1, tail = -1;
                    double at = base + upto - s;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        at += r[i];
                        if (r[i] > 0) {
                            tail = v + i;
                            if (mine < 0 && found && at > goal) mine = v + i;
                        }
                    }
                    const unsigned hit = __ballot_sync(~0u, mine >= 0), some = __ballot_sync(~0u, tail >= 0);
                    if (hit) best = __shfl_sync(~0u, mine, __ffs(hit) - 1);
                    if (some) final_one = __shfl_sync(~0u, tail, 31 - __clz(some));
                    base += __shfl_sync(~0u, upto, 31);
                }
                if (lane == 0) a.next[b] = best >= 0 ? best : final_one;
            }
        }
    }
    cluster_sync();   // (no CTA ends while another's stores are on their way to it)
}

int check_verify(const GraftVerifyParams* P) {
    clear_error();
    GRAFT_REQUIRE(P, "params pointer is null");
    GRAFT_REQUIRE(P->vocab >= 1 && P->vocab <= 0x7FFFFF00u, "vocab %u out of range", P->vocab);
    GRAFT_REQUIRE(P->tokens <= 0x03FFFFFFu, "tokens %u out of range", P->tokens);
    GRAFT_REQUIRE(P->n_seqs <= 0x00FFFFFFu, "n_seqs %u out of range", P->n_seqs);
    GRAFT_REQUIRE(P->max_tokens <= (uint32_t)kMaxTree, "max_tokens must be at most %d, not %u", kMaxTree,
                  P->max_tokens);
    GRAFT_REQUIRE(P->dtype <= GRAFT_F32, "unknown element type %u", P->dtype);
    GRAFT_REQUIRE((P->row_stride >= P->vocab && P->draft_stride >= P->vocab) || P->tokens <= 1,
                  "a row stride is below vocab");
    GRAFT_REQUIRE(P->scale >= 0x1p-100f && P->scale <= 0x1p100f && P->draft_scale >= 0x1p-100f &&
                      P->draft_scale <= 0x1p100f,
                  "scales must be positive and finite (2^-100 to 2^100)");
    return GRAFT_OK;
}

// Segments of a row: enough CTAs for several rounds over the SMs, none shorter than kMinSeg.
int segments(const GraftVerifyParams* P) {
    const uint64_t rows = P->tokens ? P->tokens : 1;
    const uint64_t want = (kRounds + rows - 1) / rows, most = std::max<uint64_t>(1, P->vocab / kMinSeg);
    return (int)std::min<uint64_t>(std::min<uint64_t>(want, most), kMaxSegs);
}

template <int DT, bool GREEDY>
int launch_verify(const VerifyArgs& a, cudaStream_t st) {
    int rc;
    if ((rc = launch_pdl("verify_drafts", verify_rows_kernel<DT, GREEDY>,
                         dim3(a.rows * (unsigned)a.segs, a.draft && !GREEDY ? 2 : 1), kRowThreads, 0, st, a)))
        return rc;
    // CTAs of a cluster: up to eight, none with less than 4096 tokens
    int ctas = 1;
    while (ctas < kMaxCluster && (uint64_t)ctas * 2 * 4096 <= a.vocab) ctas *= 2;
    const auto kern = verify_walk_kernel<DT, GREEDY>;
    if ((rc = ensure_smem((const void*)kern, sizeof(Walk)))) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.n_seqs * ctas);
    cfg.blockDim = dim3(kWalkThreads);
    cfg.dynamicSmemBytes = sizeof(Walk);
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ctas, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, ctas);
    if (e != cudaSuccess) {
        cudaGetLastError();
        set_error("verify_drafts: launch failed: %s", cudaGetErrorString(e));
        return GRAFT_ECUDA;
    }
    return check_launch("verify_drafts");
}
template <int DT>
int launch_verify(const VerifyArgs& a, cudaStream_t st) {
    return a.uniform ? launch_verify<DT, false>(a, st) : launch_verify<DT, true>(a, st);
}

}  // namespace

namespace graft {
unsigned tree_device_errors(bool clear) { return read_device_errors(g_tree_err, clear); }
}  // namespace graft

extern "C" int graft_draft_tree(const int32_t* parents, const GraftKVRange* range, uint32_t tokens,
                                uint32_t window, int32_t* mask, uint64_t mask_stride, uint32_t words,
                                int32_t* positions, graft_stream_t stream) {
    clear_error();
    GRAFT_REQUIRE(range, "range is null");
    if (range->n_seqs == 0 || tokens == 0) return GRAFT_OK;
    GRAFT_REQUIRE(range->start && range->cu_tokens && aligned(range->start, 4) && aligned(range->cu_tokens, 4),
                  "start and cu_tokens must be 4-byte aligned buffers");
    GRAFT_REQUIRE(range->n_seqs < (1u << 28) && tokens <= 0x7FFFFFFFu, "too many sequences or tokens");
    GRAFT_REQUIRE(range->max_len <= (1u << 30) && range->max_tokens <= range->max_len,
                  "max_tokens %u must not exceed max_len %u", range->max_tokens, range->max_len);
    GRAFT_REQUIRE(parents && mask && aligned(parents, 4) && aligned(mask, 4) && aligned(positions, 4),
                  "parents, mask and positions must be 4-byte aligned buffers");
    GRAFT_REQUIRE(window <= 0x7FFFFFFFu, "window %u out of range", window);
    GRAFT_REQUIRE(words >= (range->max_tokens + 31) / 32 && words <= 0x7FFFFFFFu &&
                      (mask_stride >= words || tokens <= 1),
                  "mask rows of %u words do not hold max_tokens %u", words, range->max_tokens);
    const TreeArgs a = {parents, range->start, range->cu_tokens, range->n_seqs, range->max_tokens, range->max_len,
                        tokens, window, words, (uint32_t*)mask, mask_stride, positions};
    return launch_pdl("draft_tree", draft_tree_kernel, dim3(range->n_seqs), kTreeThreads, 0, stream, a);
}

extern "C" size_t graft_verify_workspace(const GraftVerifyParams* P) {
    if (check_verify(P)) return 0;
    return std::max<size_t>(256, (size_t)2 * P->tokens * segments(P) * 8);
}

extern "C" int graft_verify_drafts(const void* logits, const void* draft, const int32_t* tokens,
                                   const int32_t* parents, const int32_t* cu_tokens, const float* uniform,
                                   const float* uniform_next, int32_t* count, int32_t* path, int32_t* next,
                                   const GraftVerifyParams* P, void* ws, size_t ws_bytes,
                                   graft_stream_t stream) {
    int rc;
    if ((rc = check_verify(P))) return rc;
    const size_t need = graft_verify_workspace(P);
    GRAFT_REQUIRE(ws && aligned(ws, 256) && ws_bytes >= need,
                  "the workspace must be 256-byte aligned and hold %zu bytes", need);
    if (P->n_seqs == 0) return GRAFT_OK;
    const size_t es = P->dtype == GRAFT_F32 ? 4 : 2;
    GRAFT_REQUIRE(cu_tokens && count && next, "cu_tokens, count and next must be given");
    if (P->tokens) {
        GRAFT_REQUIRE(logits && aligned(logits, es) && aligned(draft, es),
                      "logits and draft must be buffers aligned to their element type");
        GRAFT_REQUIRE(tokens && path, "tokens and path must be given");
    }
    GRAFT_REQUIRE(!uniform == !uniform_next, "uniform and uniform_next go together");
    GRAFT_REQUIRE(aligned(tokens, 4) && aligned(parents, 4) && aligned(cu_tokens, 4) && aligned(uniform, 4) &&
                      aligned(uniform_next, 4) && aligned(count, 4) && aligned(path, 4) && aligned(next, 4),
                  "integers and random numbers must be 4-byte aligned");
    VerifyArgs a = {};
    a.logits = logits, a.draft = uniform ? draft : nullptr, a.tokens = tokens, a.parents = parents, a.cu = cu_tokens;
    a.uniform = uniform, a.uniform_next = uniform_next;
    a.count = count, a.path = path, a.next = next;
    a.row_stride = P->row_stride, a.draft_stride = P->draft_stride;
    a.n_seqs = P->n_seqs, a.rows = P->tokens, a.max_tokens = P->max_tokens, a.vocab = P->vocab;
    a.scale = P->scale, a.draft_scale = P->draft_scale;
    a.segs = segments(P);
    a.parts = (uint64_t*)ws;
    return P->dtype == GRAFT_F16    ? launch_verify<GRAFT_F16>(a, stream)
           : P->dtype == GRAFT_BF16 ? launch_verify<GRAFT_BF16>(a, stream)
                                    : launch_verify<GRAFT_F32>(a, stream);
}
