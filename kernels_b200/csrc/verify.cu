// verify.cu -- trees of drafted tokens: their masks and positions, and which of the
// drafted tokens stand against the target's probabilities.
//
//   p = softmax(scale z), q = softmax(draft_scale z'), r = p, R = 1
//   child c accepted:  u_c q(x_c) R < r(x_c);   else  r <- max(r - R q, 0), R <- sum r
//   next = smallest v with r(v) > 0 and  sum_{w <= v} r(w) > u R
//
// Three kernels.  The first reads the rows of tokens that have children (a leaf's row matters
// only if it turns out to be the last) and leaves each segment's (reference, sum) in fp32.  The
// second walks down the tree: whether a token's first child is accepted follows from two logits
// and two sums, for all tokens at once, and so do looked-up siblings.  It goes over whole rows, in
// fp64, where a random number lies so close to a border that the sums' errors might decide, and
// where a token has several drawn children, as a cluster of CTAs a sequence.  The third spreads the
// last token's row (and the draft's, where a child was rejected) over the SMs, in fp64: cumulative
// sums decide about `next`, and at 10^5 tokens an error of 2^-24 would move one draw in a hundred to
// a neighbour.
//
// Measured (replayed): one chain of 6 tokens over 201088 17.6 us (three kernels' launches and joins),
// 10 greedily; 64 of 6 over 128256 73 us, 2.4 TB/s (the exponentials: the fp64 ones of the last rows,
// and a row is read again for its draw), 39 greedily, 82 with the draft's rows at another place in
// their 16 bytes than the target's; 16 looked-up trees of 1 to 31 over 50021 in fp32 27 us; trees of
// drawn children over 128256, 16 of 16 85 us, 64 of 64 368.  A random number next to a border, one
// sequence: 36 us more over 128256, 55 over 201088.
#include "logits.cuh"

#include <algorithm>
#include <atomic>
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
constexpr int kUnroll = 4;           // chunks of a thread's round
constexpr int kMaxSegs = 32, kMinSeg = 4096;
constexpr int kRounds = 148 * 16;    // CTAs to aim at
constexpr int kWalkThreads = 512, kWalkWarps = kWalkThreads / 32, kMaxCluster = 16;
constexpr int kDrawThreads = 256, kDrawWarps = kDrawThreads / 32, kMaxDrawSegs = 64;
constexpr float kLog2e = 1.4426950408889634f;
// The first kernel's sums are off by less than (kSumSteps + the rounds of a thread) 2^-24.  An exponent
// t = (z - ref) c is off by 3.3 2^-24 of itself (c, difference, product), its power by ln 2 of that.  A
// logit D octaves below the row's reference has powers of D + 2 kReach octaves together (its own, and
// those that follow the reference, which it may pass by kReach), and the mean D over the powers is at
// most log2 of the vocabulary, 30: 62 3.3 ln 2 < 143.  Powers: six roundings of 2^-22, 24.  Sums: 16 terms a
// round, the rounds, joins of 2, 32, 4 and 32: 31 and the rounds.
constexpr float kReach = 16.f;
constexpr int kSumSteps = 200;

struct VerifyArgs {
    const void *logits, *draft;
    const int32_t *tokens, *parents, *cu;
    const float *uniform, *uniform_next;
    int32_t *count, *path, *next;
    uint64_t row_stride, draft_stride;
    uint32_t n_seqs, rows, max_tokens, vocab;
    float scale, draft_scale;
    double off;        // how far the first kernel's sums may be off, of themselves
    int segs;
    uint64_t* parts;   // [draft: 2][rows][segs]: (reference, sum), or greedy the largest key
    // between the walk and the draw
    struct Record* records;   // [n_seqs]
    unsigned* counters;       // [n_seqs], zeroed by the walk
    int32_t* gone;            // [rows] rejected tokens of a sequence's last one, at its first row
    double* mass;             // [rows] or the masses after so many rejections
    double* sums;             // [n_seqs][draw_segs][kDrawWarps][4]
    int draw_segs;
};

// What is to be drawn from: a row without the rejected tokens (kList), or with the rejections of
// drawn children taken off (kOnce: one; kOften); greedy, the row's largest (kTop).
enum Mode : int { kDone, kList, kOnce, kOften, kTop };
struct Record {
    int mode, row, k, from;   // row of logits; rejections, and those that left nothing
    float ref, ref_q, near;   // references of the exponentials; Lp / Lq by the first kernel's sums
    double Lp, iq;            // kOften: the target's sum, and by the draft's
};

constexpr uint32_t kOrderInf = 0xFF800000u, kOrderNone = 0x007FFFFFu;   // order() of +inf and -inf
__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }
template <int DT>
constexpr int kSize = DT == GRAFT_F32 ? 4 : 2;

// The largest logit so far and the place that had it first of those taken, which are taken in their
// order; a NaN stands above all.
struct Best {
    float x = -INFINITY;
    uint32_t at = 0;
    bool nan = false;
    __device__ __forceinline__ void take(float y, uint32_t v) {
        if (!(y <= x)) {
            if (y != y) nan = true;
            else x = y, at = v;
        }
    }
    __device__ __forceinline__ uint64_t key() const {
        return nan ? ~0ull : x > -INFINITY ? key_of(x, at) : 0;
    }
};

// Elements v .. v + 7 of a row, as they lie there; those outside 0..vocab-1 are -inf and are not read.
template <int DT>
struct Eight {
    uint4 w[DT == GRAFT_F32 ? 2 : 1];
    __device__ __forceinline__ void load(const void* row, int v, int vocab) {
#pragma unroll
        for (int i = 0; i < (DT == GRAFT_F32 ? 2 : 1); ++i) {
            const int at = v + 4 * i;
            const char* p = (const char*)row + (int64_t)at * kSize<DT>;
            w[i] = at >= 0 && at + kPer<DT> <= vocab && ((uintptr_t)p & 15) == 0 ? ld_ro(p)
                                                                                 : edge_chunk<DT>(row, at, vocab);
        }
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
        if constexpr (DT == GRAFT_F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(reinterpret_cast<const uint32_t*>(w)[i]);
        } else {
            floats_of<DT>(w[0], x);
        }
    }
};

// exp(scale (x - ref)) in fp64, as 2^(t / 16): t split into a whole number n, of which n / 16 goes to
// the exponent and n % 16 takes a power from a table (16 of them have a bank each), and f in
// [-1/2, 1/2], for which 2^(f / 16) is its Chebyshev expansion on that interval up to degree 5 as a
// polynomial (off by 5e-15).
// Ten fp64 operations; the general exp costs about three times as many.  From 2^-1023 of
// exp(scale ref) down, -inf included, it is 0: however many tokens cannot come, their sum is
// nothing.  (Not for NaN.)
constexpr int kPowers = 16;
struct Expo {
    const double* pow;   // 2^(i / 16), in shared memory
    double c = 0, off = 0;
    __device__ __forceinline__ explicit Expo(const double* powers) : pow(powers) {}
    __device__ __forceinline__ void set(float r, float scale) {
        // where the next number below r has nothing, a lower slope that says so: t stays exact
        // (below the type's lowest there is none: the same step again)
        const double step = fmin((double)r - (double)__fsub_rd(r, __int_as_float(1)), 0x1p104);
        c = fmin((double)scale * (kPowers * 1.4426950408889634), 1025.0 * kPowers / step);
        off = -(double)r * c;
    }
    __device__ __forceinline__ double operator()(float x) const {
        constexpr double whole = 6755399441055744.0;   // 1.5 2^52: adding it rounds to an integer
        // t at least -1023 16 (the upper half's bits 0xC0CFF800; those of numbers below are larger), which
        // as an exponent is that of 0
        double t = fma((double)x, c, off);
        t = __hiloint2double((int)min((uint32_t)__double2hiint(t), 0xC0CFF800u), __double2loint(t));
        const double k = t + whole, f = t - (k - whole);
        const int n = __double2loint(k);
        double p = 1.2716121539285134e-09;
        p = fma(p, f, 1.4676446000606026e-07);
        p = fma(p, f, 1.3550807776365097e-05);
        p = fma(p, f, 0.0009383847924836156);
        p = fma(p, f, 0.04332169878499668);
        p = fma(p, f, 1.0000000000000044);
        const double power = pow[n & (kPowers - 1)];
        return p * __hiloint2double(__double2hiint(power) + ((n & -kPowers) << 16), __double2loint(power));
    }
};

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

// A segment of a row: a reference and the sum of exp(scale (z - it)), or the largest key.  Each
// thread has a reference of its own that moves only when a logit passes it by 2^kReach.
template <int DT, bool GREEDY>
__global__ void __launch_bounds__(kRowThreads) verify_rows_kernel(const __grid_constant__ VerifyArgs a) {
    constexpr int N = kPer<DT>, UN = kUnroll;
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
    const int off = (int)(((uintptr_t)base & 15) / kSize<DT>);   // elements before the row in its first chunk
    const int chunks = (int)(((uint64_t)off + a.vocab + N - 1) / N), per = (chunks + a.segs - 1) / a.segs;
    const int c0 = min((int)seg * per, chunks), c1 = min(c0 + per, chunks);
    // chunks that lie wholly in the row are [i0, i1)
    const int i0 = c0 + (c0 == 0 && c1 > 0 && (off || (int)a.vocab < N));
    const int i1 = max(i0, c1 - (c1 == chunks && (off + a.vocab) % N != 0));
    const float c = (of_draft ? a.draft_scale : a.scale) * kLog2e, reach = kReach / c;
    float ref = 0.f, lim = -INFINITY, L[2] = {0.f, 0.f};
    Best best;
    uint64_t key = 0;   // of what `best` took before the edge
    auto take = [&](const uint4 (&v)[UN], int ch, int step) {   // chunks ch, ch + step, ..
        if constexpr (GREEDY) {
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                float x[N];
                floats_of<DT>(v[u], x);
#pragma unroll
                for (int e = 0; e < N; ++e) best.take(x[e], (ch + u * step) * N - off + e);
            }
        } else {
            float gm = chunk_max<DT>(v[0]);
#pragma unroll
            for (int u = 1; u < UN; ++u) gm = fmaxf(gm, chunk_max<DT>(v[u]));
            if (gm > lim) {
                if (lim > -INFINITY) {
                    const float f = ex2((ref - gm) * c);
                    L[0] *= f, L[1] *= f;
                }
                ref = gm;
                lim = __fadd_rd(gm, reach);
            }
            float now[2] = {0.f, 0.f};   // (a round's sums by themselves: their errors do not grow with the row)
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    float d0, d1;
                    if constexpr (DT == GRAFT_F32) {
                        d0 = __uint_as_float(w[e]) - ref, d1 = __uint_as_float(w[e + 1]) - ref;
                    } else {
                        minus<DT>(w[e / 2], ref, d0, d1);
                    }
                    now[0] += ex2(d0 * c), now[1] += ex2(d1 * c);
                }
            }
            L[0] += now[0], L[1] += now[1];
        }
    };
    int ch = i0 + tid;
    const char* from = base + ((int64_t)ch * N - off) * kSize<DT>;
#pragma unroll 1
    for (; ch + (UN - 1) * kRowThreads < i1; ch += UN * kRowThreads, from += UN * kRowThreads * 16) {
        uint4 v[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) v[u] = ld_stream(from + u * kRowThreads * 16);
        take(v, ch, kRowThreads);
    }
    // what is left, and the row's edges (the first by thread 0, the last by thread 1), as rounds
    // with empty chunks
    const int edge = tid == 0 && i0 > c0 ? c0 : tid == 1 && i1 < c1 ? c1 - 1 : -1;
#pragma unroll 1
    for (int part = 0; part < 2; ++part) {
        if (part ? edge < 0 : ch >= i1) continue;
        // (the first edge comes after what lies behind it: joined by its place, not by its turn)
        if (GREEDY && part) key = best.key(), best = Best();
        constexpr uint32_t none = DT == GRAFT_F32 ? 0xFF800000u : DT == GRAFT_F16 ? 0xFC00FC00u : 0xFF80FF80u;
        uint4 v[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            v[u] = make_uint4(none, none, none, none);
            if (part) {
                if (u == 0) v[u] = load_chunk<DT>(base, off, a.vocab, edge);
            } else if (ch + u * kRowThreads < i1) {
                v[u] = ld_stream(from + u * kRowThreads * 16);
            }
        }
        take(v, part ? edge : ch, kRowThreads);
    }
    uint64_t* out = a.parts + ((uint64_t)of_draft * a.rows + row) * a.segs + seg;
    if constexpr (GREEDY) {
        key = max64(key, best.key());
#pragma unroll
        for (int o = 16; o; o >>= 1) key = max64(key, __shfl_xor_sync(~0u, key, o));
        if (lane == 0) sh_key[warp] = key;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < kRowWarps; ++w) key = max64(key, sh_key[w]);
            *out = key;
        }
    } else {
        // against the warp's largest reference, then the warps'
        float m = lim == -INFINITY ? -INFINITY : ref, sum = L[0] + L[1], top = m;
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        sum = m == -INFINITY ? sum : sum * ex2((m - top) * c);
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        if (lane == 0) sh[warp] = make_float2(top, sum);
        __syncthreads();
        if (tid == 0) {
            m = -INFINITY, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w) m = fmaxf(m, sh[w].x);
#pragma unroll
            for (int w = 0; w < kRowWarps; ++w)
                sum += sh[w].x == -INFINITY ? sh[w].y : sh[w].y * ex2((sh[w].x - m) * c);
            *reinterpret_cast<float2*>(out) = make_float2(m, sum);
        }
    }
}

// Which of the tokens v .. v + 7 are among k others, as bits.
__device__ __forceinline__ uint32_t among(const int* others, int k, int v) {
    uint32_t g = 0;
    for (int i = 0; i < k; ++i) {
        const uint32_t d = (uint32_t)(others[i] - v);
        if (d < 8) g |= 1u << d;
    }
    return g;
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
// The same in two halves, of which the second says that every CTA of the cluster runs.
__device__ __forceinline__ void cluster_here() {
    asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
}
__device__ __forceinline__ void cluster_all_here() {
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// Stores 64 bits at the same place of another CTA of the cluster.
__device__ __forceinline__ void store_remote(const void* at, uint32_t rank, uint64_t v) {
    asm volatile("{\n\t.reg .b32 to;\n\tmapa.shared::cluster.u32 to, %0, %1;\n\t"
                 "st.shared::cluster.b64 [to], %2;\n\t}" ::"r"(smem_u32(at)), "r"(rank), "l"(v)
                 : "memory");
}

__device__ __forceinline__ double warp_sum64(double x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    return x;
}
__device__ __forceinline__ double scan64(double x) {   // over the lanes up to this one
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(~0u, x, o);
        if ((int)(threadIdx.x & 31) >= o) x += y;
    }
    return x;
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
    uint64_t part[2][2][kMaxCluster * kWalkWarps];   // the warps' sums
    double pow[kPowers];
    double u[kMaxTree];             // random numbers
    float z[kMaxTree], zq[kMaxTree];   // logits of a token in its parent's rows
    int gone[kMaxTree], n_gone;        // rejected tokens of the current one's children
};

template <int DT, bool GREEDY>
__global__ void __launch_bounds__(kWalkThreads) verify_walk_kernel(const __grid_constant__ VerifyArgs a, int ctas) {
    extern __shared__ __align__(16) uint8_t smem[];
    Walk& sh = *reinterpret_cast<Walk*>(smem);
    // The first kernel starts this one only after its own wait, so what the caller gave is there; it is
    // read from L2, while that kernel ends.  (Without a row there is no first kernel.)
    if (a.rows == 0) pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int T = blockDim.x, W = T / 32;
    const int rank = cluster_rank(), b = blockIdx.x / ctas, NW = ctas * W;
    const int c0 = __ldcg(a.cu + b), n = __ldcg(a.cu + b + 1) - c0;
    if (c0 < 0 || n <= 0 || n > (int)a.max_tokens || (uint64_t)c0 + (uint64_t)n > a.rows) {
        pdl_wait();
        if (rank == 0 && tid == 0) a.count[b] = 0, a.next[b] = -1, a.records[b].mode = kDone;
        return;   // (the whole cluster)
    }
    if (ctas > 1) cluster_here();   // (waited for before the first store to another CTA)
    const bool drawn = !GREEDY && a.draft;
    auto row_of = [&](int i) { return (const char*)a.logits + (uint64_t)(c0 + i) * a.row_stride * kSize<DT>; };
    auto draft_of = [&](int i) { return (const char*)a.draft + (uint64_t)(c0 + i) * a.draft_stride * kSize<DT>; };
    auto usable = [](float2 s) { return s.x < INFINITY && s.y > 0.f && s.y < INFINITY; };

    // ---- the tree
    if (tid < kPowers) sh.pow[tid] = exp2(tid * (1.0 / kPowers));
    if (tid == kPowers) sh.mass[0] = 1;   // (without draft, of no token: the root's)
    for (int i = tid; i < n; i += T) {
        int p = i == 0 ? -1 : a.parents ? __ldcg(a.parents + c0 + i) : i - 1;
        p = p >= 0 && p < i ? p : -1;
        sh.parent[i] = p;
        sh.token[i] = __ldcg(a.tokens + c0 + i);
        sh.first[i] = kMaxTree;
        if constexpr (!GREEDY) sh.u[i] = __ldcg(a.uniform + c0 + i);
    }
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    for (int i = 1 + tid; i < n; i += T) {
        const int p = sh.parent[i], x = sh.token[i];
        if (p >= 0) atomicMin(&sh.first[p], i);
        if (!GREEDY && p >= 0 && (uint32_t)x < a.vocab) {   // the token's logits in its parent's rows
            sh.z[i] = logit<DT>(row_of(p), x);
            if (drawn) sh.zq[i] = logit<DT>(draft_of(p), x);
        }
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
    const int sides = drawn ? 2 : 1;
    for (int j = warp; j < n * sides; j += W) {
        const int i = drawn ? j >> 1 : j, which = drawn ? j & 1 : 0;
        if (sh.first[i] == kMaxTree) continue;
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
    __syncthreads();
    // ---- what each child's own chances say
    for (int i = 1 + tid; i < n; i += T) {
        const int p = sh.parent[i], x = sh.token[i];
        uint8_t f = kIgnored;
        bool again = false;
        double chance = 0;
        if (p >= 0 && (uint32_t)x < a.vocab) {
            if constexpr (GREEDY) {
                f = __float_as_int(sh.stat[p].x) == x ? kAccepted : kRejected;
            } else if (usable(sh.stat[p])) {
                for (int e = sh.first[p]; e != i; e = sh.sibling[e]) again |= sh.token[e] == x;
                Expo ex(sh.pow);
                ex.set(sh.stat[p].x, a.scale);
                chance = ex(sh.z[i]) / sh.stat[p].y;
                if (!drawn) {
                    f = kRejected;   // (decided below)
                } else if (usable(sh.stat_q[p])) {
                    ex.set(sh.stat_q[p].x, a.draft_scale);
                    const double uq = sh.u[i] * (ex(sh.zq[i]) / sh.stat_q[p].y);
                    f = sh.first[p] != i || fabs(uq - chance) < a.off * (uq + chance) ? kAsk
                        : uq < chance ? kAccepted : kRejected;
                }
            }
        }
        sh.flag[i] = f, sh.again[i] = again, sh.chance[i] = chance;
    }
    __syncthreads();
    if constexpr (!GREEDY) {
        if (!drawn) {
            // r is p without the earlier siblings' tokens: with L the row's sum and s that of their
            // exponentials, u (L - s) < e decides, where L alone is uncertain
            for (int i = 1 + tid; i < n; i += T)
                if (sh.flag[i] == kRejected && !sh.again[i]) {
                    double R = 1;
                    for (int e = sh.first[sh.parent[i]]; e != i; e = sh.sibling[e])
                        if (sh.flag[e] != kIgnored && !sh.again[e]) R -= sh.chance[e];
                    sh.mass[i] = R;
                }
            __syncthreads();
            for (int i = 1 + tid; i < n; i += T)
                if (sh.flag[i] == kRejected && !sh.again[i]) {
                    const double uR = sh.u[i] * sh.mass[i], e = sh.chance[i];
                    sh.flag[i] = fabs(uR - e) < a.off * sh.u[i] ? kAsk : uR < e ? kAccepted : kRejected;
                }
            __syncthreads();
        }
    }

    // ---- passes of the cluster over a row: each warp a piece of whole steps of 256 tokens
    int turn = 0;
    // every warp's values, at every CTA; value k of warp w at [k * kAll + w]
    constexpr int kAll = kMaxCluster * kWalkWarps;
    auto spread = [&](auto... v) -> const uint64_t* {
        uint64_t* to = sh.part[turn][0];
        turn ^= 1;
        int k = 0;
        if (lane < ctas)
            ((store_remote(to + k * kAll + rank * W + warp, lane, v), ++k), ...);
        cluster_sync();
        return to;
    };
    auto bits = [](double x) { return (uint64_t)__double_as_longlong(x); };
    auto value = [](uint64_t x) { return __longlong_as_double((long long)x); };
    auto total = [&](const uint64_t* parts) {   // (the same order of sums in every thread)
        double s = 0;
        for (int w = lane; w < NW; w += 32) s += value(parts[w]);
        return warp_sum64(s);
    };

    // The last token's row: exponentials, sums, rejections.
    int cur = 0, cnt = 1;
    Expo ep(sh.pow), eq(sh.pow);
    double Lp = 0, iq = 0;     // the target's sum; the draft's reciprocal sum, times Lp
    int m = 0, from = 0;       // rejections that count; those before `from` left nothing
    bool summed = false;       // Lp and iq are those of cur
    // r, times Lp, of a token with exponentials x and y, after k rejections
    auto left = [&](double x, double y, int k) {
        const double q = y * iq;
        for (int i = from; i < k; ++i) {
            const double d = sh.mass[i] * q;
            x = x > d ? x - d : 0.0;
        }
        return x;
    };
    // f of eight tokens at a time of the warp's piece of the row (and of the draft's)
    int lo = 0, hi = 0;
    auto sweep = [&](bool both, auto f) {
        const char *zp = row_of(cur), *zq = both ? draft_of(cur) : nullptr;
        const int off = (int)(((uintptr_t)zp & 15) / kSize<DT>), V = (int)a.vocab;
        const int64_t piece = (((int64_t)V + off + NW - 1) / NW + 255) / 256 * 256;
        lo = (int)min((rank * W + warp) * piece - off, (int64_t)V);
        hi = (int)min((int64_t)lo + piece, (int64_t)V);
        for (int v = lo + lane * 8; v < hi; v += 256) {
            Eight<DT> p, q;
            p.load(zp, v, V);
            if (both) q.load(zq, v, V);
            float x[8], y[8];
            p.floats(x);
            if (both) q.floats(y);
            f(x, y, v);
        }
    };
    auto sums = [&]() {        // Lp and iq
        if (summed) return;
        double sp = 0, sq = 0;
        sweep(true, [&](const float (&x)[8], const float (&y)[8], int) {
#pragma unroll
            for (int i = 0; i < 8; ++i) sp += ep(x[i]), sq += eq(y[i]);
        });
        const uint64_t* p = spread(bits(warp_sum64(sp)), bits(warp_sum64(sq)));
        Lp = total(p);
        iq = Lp / total(p + kAll);
        summed = true;
    };
    auto mass_of = [&](int k) {   // the warps' sums of r Lp after k rejections
        double s = 0;
        sweep(true, [&](const float (&x)[8], const float (&y)[8], int) {
#pragma unroll
            for (int i = 0; i < 8; ++i) s += left(ep(x[i]), eq(y[i]), k);
        });
        return spread(bits(warp_sum64(s)));
    };
    auto set_mass = [&](int k, double R) {   // (every thread has the same R)
        __syncthreads();
        if (tid == 0) sh.mass[k] = R;
        __syncthreads();
    };
    auto without = [&](int stop) {   // not drawn: the sum of p's exponentials without the tokens of
        __syncthreads();             // children that were rejected before `stop`
        if (tid == 0) sh.n_gone = 0;
        __syncthreads();
        for (int i = cur + 1 + tid; i < stop; i += T)
            if (sh.parent[i] == cur && sh.flag[i] == kRejected && !sh.again[i])
                sh.gone[atomicAdd(&sh.n_gone, 1)] = sh.token[i];
        __syncthreads();
        double s = 0;
        sweep(false, [&](const float (&x)[8], const float (&)[8], int v) {
            const uint32_t g = among(sh.gone, sh.n_gone, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) s += g >> i & 1 ? 0.0 : ep(x[i]);
        });
        return total(spread(bits(warp_sum64(s))));
    };

    if (rank == 0)
        for (int i = tid; i < n; i += T) a.path[c0 + i] = i ? -1 : c0;
    __syncthreads();
    // another CTA's shared memory may be written once that CTA runs
    if (ctas > 1) cluster_all_here();
    for (;;) {   // (every thread of the cluster takes the same way)
        int c = sh.first[cur];
        m = from = 0, summed = false;
        double swept = 0, rest = 0;   // what the row's last pass without rejected tokens gave; now left of it
        if constexpr (!GREEDY) {
            ep.set(sh.stat[cur].x, a.scale);
            if (drawn) eq.set(sh.stat_q[cur].x, a.draft_scale);
        }
        int took = -1;
        if (c < kMaxTree)
            for (; c >= 0; c = sh.sibling[c]) {
                uint8_t f = sh.flag[c];
                if (f == kIgnored) continue;
                if (!GREEDY && f == kAsk) {
                    const double u = sh.u[c];
                    const double e = ep(sh.z[c]);
                    if (drawn) {
                        sums();
                        const double q = eq(sh.zq[c]);
                        f = u * (q * iq) * sh.mass[m] < left(e, q, m) ? kAccepted : kRejected;
                    } else if (e > 0) {
                        // while the differences keep 2^-10 of the sum they are exact to 2^-42 (511 children,
                        // all rejected, over 128256: 0.2 to 0.5 ms; with a pass for each 1950 ms)
                        if (!(rest > swept * 0x1p-10)) rest = swept = without(c);
                        f = u * rest < e ? kAccepted : kRejected;
                        rest -= e;
                    } else {
                        f = kRejected;
                    }
                    if (!drawn) {
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
                // R is needed for the next child, who is asked with the whole row
                if (drawn && sh.sibling[c] >= 0) {
                    sums();
                    double R = total(mass_of(m)) / Lp;
                    if (!(R > 0)) from = m, R = 1;
                    set_mass(m, R);
                }
            }
        if (took < 0) break;
        cur = took;
        if (rank == 0 && tid == 0) a.path[c0 + cnt] = c0 + cur;
        ++cnt;
    }
    if (rank == 0 && tid == 0) a.count[b] = cnt;

    // ---- what `next` is drawn from
    if (rank == 0) {
        const bool inner = sh.first[cur] < kMaxTree;
        if constexpr (!GREEDY) {
            if (drawn) {
                for (int i = tid; i < m && m > 1; i += T) a.mass[c0 + i] = sh.mass[i];
            } else if (tid == 0 && inner) {
                m = 0;
                for (int e = sh.first[cur]; e >= 0; e = sh.sibling[e])
                    if (sh.flag[e] == kRejected && !sh.again[e]) a.gone[c0 + m++] = sh.token[e];
            }
        }
        if (tid == 0) {
            Record r = {kList, c0 + cur, m, from, 0.f, 0.f, 0.f, Lp, iq};
            if constexpr (GREEDY) {
                r.mode = inner ? kDone : kTop;
                if (inner) a.next[b] = __float_as_int(sh.stat[cur].x);
            } else if (inner && !usable(sh.stat[cur])) {
                r.mode = kDone;
                a.next[b] = -1;
            } else if (drawn && m > from) {
                r.mode = m == 1 ? kOnce : kOften;
                r.ref = sh.stat[cur].x, r.ref_q = sh.stat_q[cur].x;
                r.near = sh.stat[cur].y / sh.stat_q[cur].y;
            } else if (drawn) {
                r.k = 0;   // nothing was rejected, or nothing left: p
            }
            a.records[b] = r;
            a.counters[b] = 0;
        }
    }
    if (ctas > 1) cluster_sync();   // (no CTA ends while another's stores are on their way to it)
}

// ---- the draw
// r's sums over pieces of the row, a warp a piece; the sequence's last CTA finds the token.
template <int DT, bool GREEDY>
__global__ void __launch_bounds__(kDrawThreads, 2) verify_draw_kernel(const __grid_constant__ VerifyArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ int sh_gone[kMaxTree];
    __shared__ double sh_mass[kMaxTree], sh_pow[kPowers];
    __shared__ double sh_sum[2][kDrawWarps], sh_base;
    __shared__ float sh_x[2][9 * kDrawThreads];
    __shared__ int sh_at[kDrawWarps], sh_last, sh_owner;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int b = blockIdx.x / a.draw_segs, seg = blockIdx.x - b * a.draw_segs;
    const Record rec = a.records[b];
    if (rec.mode == kDone) return;
    const int c0 = a.cu[b], V = (int)a.vocab, NW = a.draw_segs * kDrawWarps;
    const char* zp = (const char*)a.logits + (uint64_t)rec.row * a.row_stride * kSize<DT>;
    const char* zq = (const char*)a.draft + (uint64_t)rec.row * a.draft_stride * kSize<DT>;
    const int off = (int)(((uintptr_t)zp & 15) / kSize<DT>);
    const int64_t piece = (((int64_t)V + off + NW - 1) / NW + 255) / 256 * 256;
    auto from_of = [&](int w) { return (int)min(w * piece - off, (int64_t)V); };
    const int lo = from_of(seg * kDrawWarps + warp), hi = (int)min((int64_t)lo + piece, (int64_t)V);
    double* mine = a.sums + ((uint64_t)b * NW + seg * kDrawWarps + warp) * 4;
    const double* all = a.sums + (uint64_t)b * NW * 4;

    if (tid < kPowers) sh_pow[tid] = exp2(tid * (1.0 / kPowers));
    if (rec.mode == kList)
        for (int i = tid; i < rec.k; i += kDrawThreads) sh_gone[i] = a.gone[c0 + i];
    if (rec.mode == kOften)
        for (int i = tid; i < rec.k; i += kDrawThreads) sh_mass[i] = a.mass[c0 + i];
    __syncthreads();
    Expo ep(sh_pow), eq(sh_pow);
    ep.set(rec.ref, a.scale), eq.set(rec.ref_q, a.draft_scale);
    double iq = rec.iq;
    // r, times Lp, of drawn children's rejections
    auto left = [&](double x, double y, int k) {
        const double q = y * iq;
        if (rec.mode == kOnce) return x > q ? x - q : 0.0;
        for (int i = rec.from; i < k; ++i) {
            const double d = sh_mass[i] * q;
            x = x > d ? x - d : 0.0;
        }
        return x;
    };

    // ---- the warp's piece, the next step's loads ahead
    double s0 = 0, s1 = 0, s2 = 0, s3 = 0;
    const bool both = rec.mode == kOnce || rec.mode == kOften;
    float ref = -INFINITY, lim = -INFINITY, most = -INFINITY;   // kList
    Best best;                                                  // kTop
    Eight<DT> p, q;
    auto load = [&](int v) {
        p.load(zp, v, hi);
        if (both) q.load(zq, v, hi);
    };
    if (lo < hi) load(lo + lane * 8);
    for (int v0 = lo; v0 < hi; v0 += 256) {   // (the whole warp)
        const int v = v0 + lane * 8;
        float x[8], y[8];
        p.floats(x);
        if (both) q.floats(y);
        if (v0 + 256 < hi) load(v + 256);
        if constexpr (GREEDY) {
#pragma unroll
            for (int i = 0; i < 8; ++i) best.take(x[i], v + i);
        } else if (rec.mode == kOnce) {
            // s0 - less s1: r, s2 and s3: the whole of p and q.  r is ep - less eq where that is positive,
            // less = Lp / Lq.  The first kernel's sums give that to 2 off (2^-14 for half a million tokens at
            // worst, 2^-20 as a rule), which tells the tokens where r is positive but for some whose r is below
            // that share of their p; with their sums, and the row's, one pass is enough.
            const double near = rec.near;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double e = ep(x[i]), d = eq(y[i]);
                if (e > near * d) s0 += e, s1 += d;
                s2 += e, s3 += d;
            }
        } else if (rec.mode == kOften) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double e = ep(x[i]);
                s0 += left(e, eq(y[i]), rec.k);
                s2 += e;
            }
        } else {
            // s0: what is left, s1: what is gone, against the reference s2 (the first steps' largest logit,
            // or the largest of a later step that passes it by 2^500)
            float top = x[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) top = max_nan(top, x[i]);
            most = max_nan(most, top);
            const float step = unorder(__reduce_max_sync(~0u, top == top ? order(top) : kOrderNone));
            if (step > lim) {
                const float was = ref;
                ref = step, lim = step + (float)(500.0 / (1.4426950408889634 * a.scale));
                ep.set(ref, a.scale);
                const double f = was > -INFINITY ? ep(was) : 0.0;
                s0 *= f, s1 *= f;
            }
            if (ref == -INFINITY) continue;
            const uint32_t g = rec.k ? among(sh_gone, rec.k, v) : 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double e = ep(x[i]);
                s0 += g >> i & 1 ? 0.0 : e;
                if (rec.k) s1 += g >> i & 1 ? e : 0.0;
            }
        }
    }
    if constexpr (GREEDY) {
        uint64_t key = best.key();
#pragma unroll
        for (int o = 16; o; o >>= 1) key = max64(key, __shfl_xor_sync(~0u, key, o));
        s0 = __longlong_as_double((long long)key);
    } else {
        if (!(most < INFINITY)) s0 = NAN;   // (no distribution)
        s0 = warp_sum64(s0), s1 = warp_sum64(s1);
        if (rec.mode == kList) s2 = ref;
        else s2 = warp_sum64(s2), s3 = warp_sum64(s3);
    }
    if (lane < 4) __stcg(mine + lane, lane == 0 ? s0 : lane == 1 ? s1 : lane == 2 ? s2 : s3);
    __syncthreads();
    if (tid == 0) {
        unsigned was;   // release: the CTA's sums before its count; acquire: the others'
        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(was) : "l"(a.counters + b) : "memory");
        sh_last = was + 1 == (unsigned)a.draw_segs;
    }
    __syncthreads();
    if (!sh_last) return;

    // ---- the sequence's last CTA: a thread has up to `each` pieces' sums, one after the other
    constexpr int kEach = kMaxDrawSegs * kDrawWarps / kDrawThreads;
    const int each = (NW + kDrawThreads - 1) / kDrawThreads;
    double2 in01[kEach], in23[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int w = tid * each + i;
        const bool on = i < each && w < NW;
        in01[i] = on ? __ldcg(reinterpret_cast<const double2*>(all + 4 * w)) : make_double2(0.0, 0.0);
        in23[i] = on ? __ldcg(reinterpret_cast<const double2*>(all + 4 * w + 2)) : make_double2(0.0, 0.0);
    }
    if constexpr (GREEDY) {
        uint64_t key = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) key = max64(key, (uint64_t)__double_as_longlong(in01[i].x));
#pragma unroll
        for (int o = 16; o; o >>= 1) key = max64(key, __shfl_xor_sync(~0u, key, o));
        if (lane == 0) sh_sum[0][warp] = __longlong_as_double((long long)key);
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < kDrawWarps; ++w) key = max64(key, (uint64_t)__double_as_longlong(sh_sum[0][w]));
            const uint32_t top = key >> 32;
            a.next[b] = top > kOrderNone && top < kOrderInf ? (int)(0xFFFFFFFFu - (uint32_t)key) : -1;
        }
        return;
    }
    auto sums_of = [&](double& x, double& y) {   // over the CTA
        x = warp_sum64(x), y = warp_sum64(y);
        __syncthreads();
        if (lane == 0) sh_sum[0][warp] = x, sh_sum[1][warp] = y;
        __syncthreads();
        x = y = 0;
#pragma unroll
        for (int w = 0; w < kDrawWarps; ++w) x += sh_sum[0][w], y += sh_sum[1][w];
    };
    double S[kEach];
    int k = rec.k;
    double R = 0, full = 0;
    if (rec.mode == kList) {
        float top = -INFINITY;   // (the largest of the pieces' references)
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (i < each && tid * each + i < NW) top = fmaxf(top, (float)in23[i].x);
        const uint32_t o = __reduce_max_sync(~0u, order(top));
        if (lane == 0) sh_at[warp] = (int)o;
        __syncthreads();
        uint32_t most_o = 0;
#pragma unroll
        for (int w = 0; w < kDrawWarps; ++w) most_o = max(most_o, (uint32_t)sh_at[w]);
        top = unorder(most_o);
        if (top > -INFINITY) {
            ep.set(top, a.scale);
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const double f = ep((float)in23[i].x);
                S[i] = in01[i].x * f, in23[i].x = S[i] + in01[i].y * f;
                R += S[i], full += in23[i].x;
            }
        }
    } else {
        double less = 0;
        if (rec.mode == kOnce) {
            double sq = 0;
#pragma unroll
            for (int i = 0; i < kEach; ++i) less += in23[i].x, sq += in23[i].y;
            sums_of(less, sq);
            iq = less = less / sq;
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            S[i] = fma(-less, in01[i].y, in01[i].x);
            R += S[i], full += in23[i].x;
        }
    }
    sums_of(R, full);
    int token = -1;
    // (once more with p, where nothing is left, or a rounding looked like something)
    for (bool rest_of = R > 0;; rest_of = false) {
        if (!rest_of) {
            k = 0, R = full;
#pragma unroll
            for (int i = 0; i < kEach; ++i) S[i] = in23[i].x;
        }
        if (!(R > 0 && R < INFINITY)) break;
        // ---- the piece in which the sum passes u R (none, by rounding: the last that has any)
        const double goal = (double)a.uniform_next[b] * R;
        auto before_of = [&](double x, double& whole) {   // the sum of the threads before, and of all
            const double upto = scan64(x);
            __syncthreads();
            if (lane == 31) sh_sum[0][warp] = upto;
            __syncthreads();
            double at = 0;
            whole = 0;
#pragma unroll
            for (int w = 0; w < kDrawWarps; ++w) {
                if (w < warp) at += sh_sum[0][w];
                whole += sh_sum[0][w];
            }
            return at + (upto - x);
        };
        double mass = 0, whole;
#pragma unroll
        for (int i = 0; i < kEach; ++i) mass += S[i];
        if (tid == 0) sh_owner = 0x7FFFFFFF, sh_last = -1;
        double at = before_of(mass, whole);
        int owner = 0x7FFFFFFF, last = -1;
        double start = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (S[i] > 0) {
                last = tid * each + i;
                if (owner == 0x7FFFFFFF && at + S[i] > goal) owner = last, start = at;
            }
            at += S[i];
        }
        if (owner != 0x7FFFFFFF) atomicMin(&sh_owner, owner);
        if (last >= 0) atomicMax(&sh_last, last);
        __syncthreads();
        const bool found = sh_owner != 0x7FFFFFFF;
        if (found && owner == sh_owner) sh_base = start;
        __syncthreads();
        start = found ? sh_base : 0;
        owner = found ? sh_owner : sh_last;
        // ---- the token: up to eight a thread, from shared memory (in loops of two: one CTA a sequence
        // comes here, and its instructions come from far).  Pass 0: the piece's first that passes u R; 1: its
        // last that has any.  Sums and differences round, so that a piece may have a sum and no such token:
        // then the first that has any of the pieces behind, or else the last of those before.
        const bool two = both && k;
        auto place = [](int i) { return i + (i >> 3); };
        const int behind = found ? NW - 1 - owner : 0;
#pragma unroll 1
        for (int pass = found ? 0 : 1; token < 0; ++pass) {
            const bool tail = pass == 1 || pass - 2 >= behind;
            const int piece_of = pass < 2 ? owner : tail ? owner - 1 - (pass - 2 - behind) : owner + pass - 1;
            if (piece_of < 0) break;
            const double past = pass < 2 ? goal : -1;
            const int first = from_of(piece_of), end = (int)min((int64_t)first + piece, (int64_t)V);
            const int per = min(8, (end - first + 2 * kDrawThreads - 1) / (2 * kDrawThreads) * 2);   // tokens of a thread
            double base = pass < 2 ? start : 0;
            int late = -1;
#pragma unroll 1
            for (int v0 = first; v0 < end && token < 0; v0 += per * kDrawThreads) {
                float x[8], y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int v = v0 + i * kDrawThreads + tid;
                    const bool in = i < per && v >= 0 && v < end;
                    x[i] = in ? logit<DT>(zp, v) : -INFINITY;
                    y[i] = in && two ? logit<DT>(zq, v) : -INFINITY;
                }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < per) {
                        sh_x[0][place(i * kDrawThreads + tid)] = x[i];
                        sh_x[1][place(i * kDrawThreads + tid)] = y[i];
                    }
                __syncthreads();
                const int v = v0 + per * tid;
                const uint32_t g = !both && k ? among(sh_gone, k, v) : 0;
                auto rest = [&](int i, double& r0, double& r1) {   // of tokens v + i and the next
                    const int at = per * tid + i;
                    r0 = ep(sh_x[0][place(at)]), r1 = ep(sh_x[0][place(at + 1)]);
                    if (two) r0 = left(r0, eq(sh_x[1][place(at)]), k), r1 = left(r1, eq(sh_x[1][place(at + 1)]), k);
                    r0 = g >> i & 1 ? 0.0 : r0, r1 = g >> i & 2 ? 0.0 : r1;
                };
                double s = 0;
#pragma unroll 1
                for (int i = 0; i < per; i += 2) {
                    double r0, r1;
                    rest(i, r0, r1);
                    s += r0 + r1;
                }
                double before = base + before_of(s, whole);
                int here = tail ? -1 : 0x7FFFFFFF;
                if (tail || before + s > past) {
#pragma unroll 1
                    for (int i = 0; i < per; i += 2) {
                        double r[2];
                        rest(i, r[0], r[1]);
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            before += r[j];
                            if (r[j] > 0) {
                                if (tail) here = v + i + j;
                                else if (before > past) here = min(here, v + i + j);
                            }
                        }
                    }
                }
                here = tail ? __reduce_max_sync(~0u, here) : __reduce_min_sync(~0u, here);
                if (lane == 0) sh_at[warp] = here;
                __syncthreads();
                for (int w = 0; w < kDrawWarps; ++w) here = tail ? max(here, sh_at[w]) : min(here, sh_at[w]);
                if (tail) late = max(late, here);
                else if (here != 0x7FFFFFFF) token = here;
                base += whole;
                __syncthreads();
            }
            if (tail) token = late;
        }
        if (token >= 0 || !rest_of) break;
    }
    if (tid == 0) a.next[b] = token;
}

int check_verify(const GraftVerifyParams* P) {
    clear_error();
    GRAFT_REQUIRE(P, "params pointer is null");
    GRAFT_REQUIRE(P->vocab >= 1 && P->vocab <= 1u << 30, "vocab %u out of range", P->vocab);
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

// Segments of a row: enough CTAs for several rounds over the SMs (counted as 148, for the workspace is
// sized before there is a device), none shorter than kMinSeg.
int segments(const GraftVerifyParams* P) {
    const uint64_t rows = P->tokens ? P->tokens : 1;
    const uint64_t want = (kRounds + rows - 1) / rows, most = std::max<uint64_t>(1, P->vocab / kMinSeg);
    return (int)std::min<uint64_t>(std::min<uint64_t>(want, most), kMaxSegs);
}

// CTAs that go over a sequence's last row: two rounds of two an SM, none with less than 2048 tokens.
int draw_segments(const GraftVerifyParams* P) {
    const uint64_t seqs = P->n_seqs ? P->n_seqs : 1;
    const uint64_t want = std::max<uint64_t>(1, 148 * 4 / seqs), most = std::max<uint64_t>(1, P->vocab / 2048);
    return (int)std::min<uint64_t>(std::min<uint64_t>(want, most), kMaxDrawSegs);
}

// The workspace's parts; its size.
size_t carve(const GraftVerifyParams* P, char* ws, VerifyArgs* a) {
    size_t at = 0;
    auto take = [&](size_t bytes) {
        char* p = ws + at;
        at += (bytes + 255) / 256 * 256;
        return p;
    };
    const size_t rows = P->tokens, seqs = P->n_seqs;
    char* parts = take(2 * rows * segments(P) * 8);
    char* records = take(seqs * sizeof(Record));
    char* counters = take(seqs * 4);
    char* gone = take(rows * 4);
    char* mass = take(rows * 8);
    char* sums = take(seqs * draw_segments(P) * kDrawWarps * 32);
    if (a) {
        a->parts = (uint64_t*)parts, a->records = (Record*)records, a->counters = (unsigned*)counters;
        a->gone = (int32_t*)gone, a->mass = (double*)mass, a->sums = (double*)sums;
    }
    return std::max<size_t>(256, at);
}

template <int DT, bool GREEDY>
int launch_verify(const VerifyArgs& a, cudaStream_t st) {
    int rc = GRAFT_OK;
    if (a.rows)   // (without a row, every sequence is without tokens)
        rc = launch_pdl("verify_drafts", verify_rows_kernel<DT, GREEDY>,
                        dim3(a.rows * (unsigned)a.segs, a.draft && !GREEDY ? 2 : 1), kRowThreads, 0, st, a);
    if (rc) return rc;
    DeviceInfo di;
    if ((rc = current_device_info(&di))) return rc;
    // Whole rows are gone over during the walk where a token may have several drawn children: then a
    // cluster a sequence (sixteen CTAs while all have an SM of their own), no CTA of it with less
    // than 4096 tokens.
    int ctas = 1;
    if (!GREEDY && a.draft && a.parents) {
        const int most = (uint64_t)a.n_seqs * kMaxCluster <= (uint64_t)di.sm_count ? kMaxCluster : kMaxCluster / 2;
        while (ctas < most && (uint64_t)ctas * 2 * 4096 <= a.vocab) ctas *= 2;
    }
    const auto kern = verify_walk_kernel<DT, GREEDY>;
    if ((rc = ensure_smem((const void*)kern, sizeof(Walk)))) return rc;
    static std::atomic<uint64_t> wide{0};   // devices where clusters of sixteen are allowed
    const uint64_t bit = 1ull << (di.device & 63);
    if (ctas > 8 && !(wide.load(std::memory_order_relaxed) & bit)) {
        GRAFT_CUDA(cudaFuncSetAttribute((const void*)kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        wide.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.n_seqs * ctas);
    cfg.blockDim = dim3(kWalkThreads);
    cfg.dynamicSmemBytes = sizeof(Walk);
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    int attrs = 0;
    if (ctas > 1) {
        at[attrs].id = cudaLaunchAttributeClusterDimension;
        at[attrs].val.clusterDim.x = ctas, at[attrs].val.clusterDim.y = 1, at[attrs].val.clusterDim.z = 1;
        ++attrs;
    }
    if (pdl_enabled()) {
        at[attrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[attrs].val.programmaticStreamSerializationAllowed = 1;
        ++attrs;
    }
    cfg.attrs = at;
    cfg.numAttrs = attrs;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, ctas);
    if (e != cudaSuccess) {
        cudaGetLastError();
        set_error("verify_drafts: launch failed: %s", cudaGetErrorString(e));
        return GRAFT_ECUDA;
    }
    if ((rc = check_launch("verify_drafts"))) return rc;
    return launch_pdl("verify_drafts", verify_draw_kernel<DT, GREEDY>, dim3(a.n_seqs * (unsigned)a.draw_segs),
                      kDrawThreads, 0, st, a);
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
    return carve(P, nullptr, nullptr);
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
    GRAFT_REQUIRE(!P->tokens || !uniform == !uniform_next, "uniform and uniform_next go together");
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
    a.segs = segments(P), a.draw_segs = draw_segments(P);
    const uint64_t round = (uint64_t)kUnroll * kRowThreads * (16 / es);   // tokens of a CTA's round
    a.off = (kSumSteps + (double)((a.vocab / a.segs + round - 1) / round + 2)) * 0x1p-24;
    carve(P, (char*)ws, &a);
    return P->dtype == GRAFT_F16    ? launch_verify<GRAFT_F16>(a, stream)
           : P->dtype == GRAFT_BF16 ? launch_verify<GRAFT_BF16>(a, stream)
                                    : launch_verify<GRAFT_F32>(a, stream);
}
