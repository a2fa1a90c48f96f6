// attn_cols.cuh -- attention over the 8-bit cache for 17 to 64 query rows a head (33 to 64 for heads of
// up to 64 dims; trees of a few drafted tokens), on the fifth-generation tensor cores with the rows as columns.
//
// The matrix unit's 128 rows are keys, then dims; the query rows are its N = 64 columns:
//   S^T [128 keys x 64]  = K [128 x D] q^T          (K from shared memory, K-major)
//   O^T [dims x 64]     += V^T [dims x 128 keys] P  (V as it lies there: M-major, P by softmax)
// so a call pays for the exponentials of the rows that it has, where the kernel for many rows
// (attn_chunk.cuh) pays for 256.  A CTA (one per SM) works on units of 128 keys in these roles:
//   softmax     (two groups of 4 warps)  thread = key = TMEM lane: reads the key's scores, takes the
//               weights and stores them as fp16 in shared memory (a row of 128 bytes a key, the
//               N-major B operand of the second product).  Up to 32 rows: the groups take every other
//               unit; more: 32 rows of every unit each;
//   loader      (one warp)  bulk copies of a unit's codes to shared memory, some units ahead (bytes in
//               flight are what HBM asks for);
//   converters  (2 warps for K, 2 for V)  codes to fp16 stages, 128-byte swizzled rows of 64 dims: the
//               K-major A operand of the first product and, unchanged in layout, the M-major A
//               operand of the second;
//   MMA         (one lane).
// A key's scales are numbers of its thread.  A group has its own references (by row, in shared
// memory) and sums (of its keys, in registers), and where the groups take turns its own output; these
// are joined at the end of a piece.  A reference follows a row's maximum only when a score passes it by
// more than kPSlack: every thread says so at the one barrier that a unit has, and then the group looks
// for the maxima.  What runs once a piece is kept in short loops: its instructions are not at hand.
// With head_dim up to 64 the second product's other 64 dims are whatever lies behind V; nothing is
// read of them.
//
// What bounds it: the softmax of a unit is a chain of about 2500 cycles (scores from tensor memory 60,
// references and check 750, weights 1200, stores and their fence 300), which two groups halve; the
// converters of 128 dims in e4m3 take 1300 for a unit, shared memory's bandwidth 1800.  32 requests of
// 8 tokens and up to 8191 keys, 32 query heads on 8 of 128, e4m3: 124 us, 2.2 TB/s; the many-row
// kernel takes 238.  A piece of a pair costs about five units more.  Codes that converters read
// ahead into registers, or eight converter warps, were slower (140 us and more).
#pragma once
#include "attn_chunk.cuh"

namespace graft {
namespace dev {

template <int DP>
struct Cols {
    static constexpr int KT = 128;                   // keys of a unit
    static constexpr int N = 64;                     // columns
    static constexpr int ST = DP <= 64 ? 2 : 1;      // stages of fp16 K and V
    static constexpr int RAW = DP <= 64 ? 6 : 3;     // units of codes that are copied or on their way
    static constexpr int GROUPS = 2, SOFT = 4 * GROUPS, CONV = 4;
    static constexpr int THREADS = 32 * (SOFT + CONV + 2);   // (and MMA, loader)
    static constexpr int DB = DP / 64;               // blocks of 64 dims
    static constexpr int Q_BYTES = DB * N * 128;
    static constexpr int KV_BYTES = DB * KT * 128;   // K or V of a unit
    static constexpr int P_BYTES = KT * 128;         // weights of a unit
    static constexpr int CODES = DP * KT;            // codes of K or V of a unit
    static constexpr int SMEM = 1024 + Q_BYTES + 2 * ST * KV_BYTES + GROUPS * P_BYTES + 2 * RAW * CODES;
    static constexpr int SC = 8;                     // slots of a unit's scales (up to ST + AHEAD + 1 in use)
    static constexpr int S_BUFS = 4;                 // scores in tensor memory
    static constexpr int AHEAD = 2;                  // units whose scores are begun before the first one's product
    static constexpr int O_COL = S_BUFS * N;         // its outputs behind them (one a group that takes turns)
    // floats of a partial result: O row by row, reference and sum of each row
    static constexpr int PARTIAL = N * DP + 2 * N;
};

// Lane l's result: row l's value over all lanes, of 32 rows that each lane has (op: max or sum).
template <typename Op>
__device__ __forceinline__ float reduce_rows(float (&v)[32], Op op) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int half = 16; half > 0; half >>= 1) {
        const bool up = lane & half;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const float mine = up ? v[i + half] : v[i], other = up ? v[i] : v[i + half];
            v[i] = op(mine, __shfl_xor_sync(~0u, other, half));
        }
    }
    return v[0];
}

__device__ __forceinline__ void tmem_ld8(uint32_t addr, uint32_t (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr),
                 "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

template <int DP, int NR, int FMT>   // NR: rows, up to 32 or 64
__global__ void __launch_bounds__(Cols<DP>::THREADS, 1)
    attn_cols_kernel(const __grid_constant__ AttnArgs a, unsigned* err) {
    using C = Cols<DP>;
    constexpr int KT = C::KT, ST = C::ST, SC = C::SC, N = C::N;
    constexpr bool TURNS = NR == 32;   // the groups take turns
    struct Walk {
        int at, prefix;   // next unit, units before the sequence
        Seq s;
        int b, nu, u0;    // sequence, its units a head with the pad (0: none), its first unit
        int h, lo, hi;    // the piece: head, units [lo, hi)
        int p0;           // first unit of the pair
    };
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Walk sh_edge[2];
    __shared__ uint64_t kfull[ST], kfree[ST], vfull[ST], vfree[ST], scfull[SC], qfull, done;
    __shared__ uint64_t rawfull[C::RAW], rawfree[C::RAW];
    __shared__ uint64_t sfull[C::S_BUFS], pfull[2], pdone[2];   // (weights: by the unit's parity)
    __shared__ float4 scales[SC][KT / 16];            // k_scale, log2(v_scale), 1 / v_scale
    __shared__ float raw_scales[C::RAW][2][KT / 16];
    // a group's 32 rows: scale log2(e) and reference; what a moved reference makes of earlier weights;
    // the warps' maxima, then sums
    __shared__ float2 cm[C::GROUPS][32];
    __shared__ float grow[C::GROUPS][32], part[C::GROUPS][4][32];
    __shared__ float4 joined[N];                      // of a row: reference, sum, factors of the groups
    __shared__ int first[N];                          // of a token: the first key that it sees,
    __shared__ uint32_t sh_mask[N][2];                // and the new ones
    __shared__ uint32_t tmem_at;
    __shared__ volatile int dead;                     // a wait gave up: every role stops
    __shared__ int sh_scan[C::THREADS / 32], sh_pairs[C::THREADS / 32];
    __shared__ int sh_last;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int D = a.dim, H = a.heads, G = a.group;
    uint8_t* base = smem + ((1024 - (smem_u32(smem) & 1023)) & 1023);
    uint8_t *sq = base, *sk = base + C::Q_BYTES, *sv = sk + ST * C::KV_BYTES, *sp = sv + ST * C::KV_BYTES;
    uint8_t* raw = sp + C::GROUPS * C::P_BYTES;   // [RAW][K, V][key][dim]
    if (tid == 0) {
        for (int i = 0; i < ST; ++i) {   // (full: converter warps; free: commits)
            mbar_init(smem_u32(&kfull[i]), C::CONV / 2), mbar_init(smem_u32(&vfull[i]), C::CONV / 2);
            mbar_init(smem_u32(&kfree[i]), 1), mbar_init(smem_u32(&vfree[i]), 1);
        }
        for (int i = 0; i < SC; ++i) mbar_init(smem_u32(&scfull[i]), 1);
        for (int i = 0; i < C::RAW; ++i)   // (the loader's lanes' copies of scales, and its count of bytes)
            mbar_init(smem_u32(&rawfull[i]), 17), mbar_init(smem_u32(&rawfree[i]), C::CONV);
        for (int i = 0; i < C::S_BUFS; ++i) mbar_init(smem_u32(&sfull[i]), 1);      // commits
        for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&pfull[i]), TURNS ? 4 : 8), mbar_init(smem_u32(&pdone[i]), 1);
        mbar_init(smem_u32(&qfull), C::SOFT);
        mbar_init(smem_u32(&done), 1);
        dead = 0;
    }
    fence_mbar_init();
    pdl_wait();
    pdl_launch_dependents();

    // ---- units of every sequence: their total, and where this CTA's bounds lie
    auto open_seq = [&](Walk& w) {
        w.s = load_seq(a, w.b, err);
        w.u0 = first_key(a, w.s.start) / KT;
        w.nu = w.s.n ? (w.s.start + w.s.n + KT - 1) / KT - w.u0 + a.pad_units : 0;
    };
    Split<int> split;
    Walk cw;
    int fe;   // this CTA's units: [cw.at, fe)
    {
        int U = 0, pairs = 0, prefix = 0;
        auto scan = [&](uint32_t b0, int from) {
            cw.b = b0 + tid, cw.nu = 0;
            if (cw.b < (int)a.n_seqs) open_seq(cw);
            int x = cw.nu;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(~0u, x, o);
                if (lane >= o) x += y;
            }
            const int some = __popc(__ballot_sync(~0u, cw.nu > 0));
            __syncthreads();
            if (lane == 31) sh_scan[warp] = x, sh_pairs[warp] = some;
            __syncthreads();
            prefix = from + x - cw.nu;
            int total = 0;
            for (int w = 0; w < C::THREADS / 32; ++w) {
                const int y = sh_scan[w];
                if (w < warp) prefix += y;
                total += y, pairs += sh_pairs[w];
            }
            return total;
        };
        for (uint32_t b0 = 0; b0 < a.n_seqs; b0 += C::THREADS) U += scan(b0, 0);
        U *= H, pairs *= H;
        if (U == 0) return;
        const int grid = min((int)gridDim.x, max(pairs, (U - pairs * a.pad_units) / a.min_units));
        if ((int)blockIdx.x >= grid) return;
        split.set(U, grid, a.pad_units, a.min_units);
        const int x0 = split.bound(blockIdx.x), x1 = split.bound(blockIdx.x + 1);
        int from = 0;
        for (uint32_t b0 = 0; b0 < a.n_seqs; b0 += C::THREADS) {
            if (a.n_seqs > C::THREADS) from += scan(b0, from);   // (else all is still at hand)
            cw.prefix = prefix * H;
            const int e = cw.prefix + cw.nu * H;
            if (cw.prefix <= x0 && x0 < e) sh_edge[0] = cw;
            if (cw.prefix <= x1 && x1 < e) sh_edge[1] = cw;
        }
        __syncthreads();
        auto edge = [&](const Walk& w, int x) {
            const int p0 = w.prefix + (x - w.prefix) / w.nu * w.nu;
            return split.snapped(x, p0, p0 + w.nu);
        };
        fe = x1 >= U ? U : edge(sh_edge[1], x1);
        cw = sh_edge[0];
        cw.at = edge(cw, x0);
        if (cw.at >= fe) return;
    }
    auto next_piece = [&](Walk& w) {   // false: no more
        if (w.at >= fe) return false;
        while (w.at >= w.prefix + w.nu * H) {
            w.prefix += w.nu * H;
            ++w.b;
            open_seq(w);
        }
        w.h = (w.at - w.prefix) / w.nu;
        w.p0 = w.prefix + w.h * w.nu;
        const int e = min(fe, w.p0 + w.nu);
        w.lo = w.u0 + max(0, w.at - w.p0 - a.pad_units);
        w.hi = w.u0 + e - w.p0 - a.pad_units;
        w.at = e;
        return true;
    };
    // Waits as in the kernel for many rows: bounded; after one gave up none waits.
    auto late = [&](uint64_t& t0) {
        if (dead) return true;
        const uint64_t now = global_ns();
        if (t0 == 0) t0 = now;
        if (now - t0 <= kAttnWaitNs) return false;
        atomicOr(err, (unsigned)GRAFT_KV_EWAIT);
        dead = 1;
        return true;
    };
    auto wait = [&](uint64_t* bar, uint32_t phase) {
        if (mbar_test(smem_u32(bar), phase & 1)) return;   // (the usual case)
        uint64_t t0 = 0;
        while (!mbar_try_wait(smem_u32(bar), phase & 1))
            if (late(t0)) break;
    };
    auto spin = [&](uint64_t* bar, uint32_t phase) {
        uint64_t t0 = 0;
        for (uint32_t i = 1; !mbar_test(smem_u32(bar), phase & 1); ++i)
            if ((i & 255) == 0 && late(t0)) break;
    };
    if (warp == C::SOFT + C::CONV) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&tmem_at)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // weights of columns that no row has stay 0
    for (int i = tid; i < C::GROUPS * C::P_BYTES / 16; i += C::THREADS)
        reinterpret_cast<uint4*>(sp)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
    tc5_fence_before();
    __syncthreads();
    tc5_fence_after();
    const uint32_t tmem = tmem_at;

    if (warp < C::SOFT) {
        // =========================================================== softmax
        // (registers move from the converters: 8 x 152 + 4 x 80 = 12 x 128)
        asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
        const int g = warp >> 2, key = (warp & 3) * 32 + lane;   // key of the unit = TMEM lane
        const uint32_t tlane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const int row0 = TURNS ? 0 : 32 * g;                     // the group's first row
        const uint32_t to = tlane + C::O_COL + (TURNS ? g * N : row0);
        auto group_sync = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory"); };
        auto both_sync = [&]() { asm volatile("bar.sync 3, 256;" ::: "memory"); };
        int it = 0;   // units done by the CTA
        while (next_piece(cw)) {
            const int R = cw.s.n * G;
            // ---- the rows' queries as fp16: four threads a row
            {
                const int r = tid >> 2, tok = r / G, hq = cw.h * G + r - tok * G;
                const bool on = r < R;
                const uint16_t* src = (const uint16_t*)a.q + (size_t)(cw.s.c0 + (on ? tok : 0)) * a.q_tok +
                                      (size_t)(on ? hq : 0) * a.q_head;
                uint4 x[DP / 32];   // chunks q, q + 4, ..
                float amax = 0.f;
#pragma unroll
                for (int c = 0; c < DP / 32; ++c) {
                    const int d = 8 * ((tid & 3) + 4 * c);
                    x[c] = make_uint4(0, 0, 0, 0);
                    if (on && d < D) x[c] = *reinterpret_cast<const uint4*>(src + d);
                    if (a.bf16) {
                        const uint32_t w[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 p = unpack2<GRAFT_BF16>(w[e]);
                            // (a NaN must not hide behind fmaxf)
                            amax = (p.x == p.x) ? fmaxf(amax, fabsf(p.x)) : INFINITY;
                            amax = (p.y == p.y) ? fmaxf(amax, fabsf(p.y)) : INFINITY;
                        }
                    }
                }
                float down = 1.f, up = 1.f;
                if (a.bf16) {
                    amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
                    amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
                    const float e = bf16_row_exponent(amax);
                    down = exp2f(-e), up = exp2f(e);
                }
#pragma unroll
                for (int c = 0; c < DP / 32; ++c) {
                    uint32_t w[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (a.bf16) {
                            const float2 p = unpack2<GRAFT_BF16>(w[e]);
                            w[e] = pack_h2(p.x * down, p.y * down);
                        }
                    const int at = (tid & 3) + 4 * c;   // chunk of 8 dims
                    *reinterpret_cast<uint4*>(sq + ((at >> 3) * N + r) * 128 + (((at & 7) ^ (r & 7)) << 4)) =
                        make_uint4(w[0], w[1], w[2], w[3]);
                }
                if ((tid & 3) == 0) {
                    // (columns without a row have no weights: their reference is out of reach)
                    const float2 v = make_float2(on ? a.scale * kLog2e * up : 0.f, on ? kNoMax : -kNoMax);
                    if (!TURNS) cm[r >> 5][r & 31] = v;
                    else if (r < 32) cm[0][r] = v, cm[1][r] = v;
                }
                if (tid < cw.s.n) first[tid] = first_tree_key(a, cw.s, tid);
                if (tid < 2 * cw.s.n && 32 * (tid & 1) < cw.s.n)
                    sh_mask[tid >> 1][tid & 1] = a.mask[(size_t)(cw.s.c0 + (tid >> 1)) * a.mask_stride + (tid & 1)];
                fence_proxy_async_smem();
                tc5_fence_before();   // (the last piece's O has been read)
                both_sync();
                if (lane == 0) mbar_arrive(smem_u32(&qfull));
            }
            const int len = cw.s.start + cw.s.n;
            float l[32];   // sums of this key's weights
#pragma unroll
            for (int r = 0; r < 32; ++r) l[r] = 0.f;
            int before = -1;   // the group's last unit
            for (int u = cw.lo; u < cw.hi; ++u, ++it) {
                if (TURNS && (it & 1) != g) continue;
                const int j = u * KT + key;
                // which rows see the key
                uint64_t see = ~0ull;
                const bool careful = a.window || (u + 1) * KT > cw.s.start;
                if (careful) {
                    see = 0;
                    const int i = j - cw.s.start;
                    const uint64_t rows = (G >= 64 ? 0 : 1ull << G) - 1;
                    if (i < 0) {
                        for (int t = 0; t < cw.s.n; ++t)
                            if (j >= first[t]) see |= rows << (t * G);
                    } else if (j < len) {
                        for (int t = 0; t < cw.s.n; ++t)
                            if (sh_mask[t][i >> 5] >> (i & 31) & 1u)
                                see |= rows << (t * G);
                    }
                }
                wait(&scfull[it % SC], it / SC);
                const float4 sc = scales[it % SC][key >> 4];   // k_scale, log2(v_scale), 1 / v_scale
                wait(&sfull[it & 3], it >> 2);
                tc5_fence_after();
                float t[32];
                tmem_ld32(tlane + (it & 3) * N + row0, reinterpret_cast<uint32_t(&)[32]>(t));
                tmem_wait_ld();
                const uint32_t seen = (uint32_t)(see >> row0);
                float over = -INFINITY;
#pragma unroll
                for (int r = 0; r < 32; r += 2) {
                    const float4 v = *reinterpret_cast<const float4*>(&cm[g][r]);
                    unpair(fma2(pair(t[r], t[r + 1]), mul2(pair(v.x, v.z), pair(sc.x, sc.x)), pair(sc.y, sc.y)),
                           t[r], t[r + 1]);
                    if (careful) {
                        t[r] = seen >> r & 1 ? t[r] : -INFINITY;
                        t[r + 1] = seen >> (r + 1) & 1 ? t[r + 1] : -INFINITY;
                    }
                    over = fmaxf(over, fmaxf(t[r] - v.y, t[r + 1] - v.w));
                }
                uint32_t move;
                asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
                             "barrier.cta.red.or.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                             : "=r"(move) : "r"((uint32_t)(over > kPShift + kPSlack)), "r"(1 + g) : "memory");
                if (move) {   // ---- the references follow the rows' maxima
                    {
                        float v[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = t[i];
                        part[g][warp & 3][lane] = reduce_rows(v, [](float x, float y) { return fmaxf(x, y); });
                    }
                    group_sync();
                    if (key < 32) {
                        const float mx = fmaxf(fmaxf(part[g][0][key], part[g][1][key]),
                                               fmaxf(part[g][2][key], part[g][3][key]));
                        const float was = cm[g][key].y, now = fmaxf(was, reference(mx, kPShift));
                        grow[g][key] = ex2(was - now);
                        cm[g][key].y = now;
                    }
                    group_sync();
#pragma unroll
                    for (int r = 0; r < 32; ++r) l[r] *= grow[g][r];
                    if (before >= 0) {   // the output, once the product before has been added
                        wait(&pdone[before & 1], before >> 1);
                        tc5_fence_after();
#pragma unroll 1
                        for (int c = 0; c < 4; ++c) {
                            uint32_t v[8];
                            tmem_ld8(to + 8 * c, v);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * grow[g][8 * c + e]);
                            tmem_st8(to + 8 * c, v);
                        }
                        tmem_wait_st();
                    }
                }
                // ---- the weights: 2^(t - m), times what v_scale undoes in their sums
#pragma unroll
                for (int r = 0; r < 32; r += 2) {
                    const float4 v = *reinterpret_cast<const float4*>(&cm[g][r]);
                    t[r] = ex2(t[r] - v.y), t[r + 1] = ex2(t[r + 1] - v.w);
                    l[r] = fmaf(t[r], sc.z, l[r]), l[r + 1] = fmaf(t[r + 1], sc.z, l[r + 1]);
                }
                if (it > 1) wait(&pdone[it & 1], (it >> 1) - 1);   // (the product before has read the weights)
                uint8_t* prow = sp + (it & 1) * C::P_BYTES + key * 128;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    *reinterpret_cast<uint4*>(prow + ((((row0 >> 3) + k) ^ (key & 7)) << 4)) =
                        make_uint4(pack_h2(t[8 * k], t[8 * k + 1]), pack_h2(t[8 * k + 2], t[8 * k + 3]),
                                   pack_h2(t[8 * k + 4], t[8 * k + 5]), pack_h2(t[8 * k + 6], t[8 * k + 7]));
                fence_proxy_async_smem();
                tc5_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&pfull[it & 1]));
                before = it;
            }
            // ---- the group's sums; its output once its last product is there
            part[g][warp & 3][lane] = reduce_rows(l, [](float x, float y) { return x + y; });
            if (before >= 0) wait(&pdone[before & 1], before >> 1);
            tc5_fence_after();
            both_sync();
            // ---- joined: reference, sum, and the factors of the groups' outputs, by row
            const bool other = TURNS && cw.hi - cw.lo > 1;   // both groups had units of these rows
            const int only = (it - 1) & 1;                   // else the one that had
            if (tid < NR) {
                const int i = tid & 31;
                auto of = [&](int k) { return make_float2(cm[k][i].y, part[k][0][i] + part[k][1][i] + part[k][2][i] + part[k][3][i]); };
                if (other) {
                    const float2 p = of(0), q = of(1);
                    const float M = fmaxf(p.x, q.x), f0 = ex2(p.x - M), f1 = ex2(q.x - M);
                    joined[tid] = make_float4(M, p.y * f0 + q.y * f1, f0, f1);
                } else {
                    const float2 p = of(TURNS ? only : tid >> 5);
                    joined[tid] = make_float4(p.x, p.y, 1.f, 1.f);
                }
            }
            both_sync();
            // ---- the outputs go to shared memory, [row][dim], where groups that take turns are added up
            // (O^T has the dims as lanes: warps 0 and 1 of a group, all four for more than 64 dims)
            float* sum = reinterpret_cast<float*>(sp);   // (the weights have been read)
#pragma unroll 1
            for (int turn = TURNS ? 1 : 0; turn >= 0; --turn) {
                if ((!TURNS || g == turn) && before >= 0 && (DP > 64 || (warp & 3) < 2)) {
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t o[8];
                        tmem_ld8(to + 8 * c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int r = row0 + 8 * c + e;
                            const float f = g ? joined[r].w : joined[r].z;
                            float* at = &sum[r * DP + key];
                            const float x = __uint_as_float(o[e]) * f;
                            *at = turn == 0 && other ? *at + x : x;
                        }
                    }
                }
                both_sync();
            }
            // ---- two dims of a row at a time: the output, or the piece's part of a cut pair
            constexpr int HALF = DP / 2, STEP = 32 * C::SOFT / HALF;
            const int r0 = tid / HALF, d = 2 * (tid % HALF);
            auto finish = [&](int r, float2 x, float M, float L) {   // x, L relative to 2^M
                if (d >= D) return;
                const int tok = r / G, hq = cw.h * G + r - tok * G;
                float ref = M, fo = 1.f;
                if (a.sinks) {
                    const float sk = a.sinks[hq] * kLog2e;
                    if (sk > ref) {
                        fo = ex2(ref - sk);
                        L = L * fo + 1.f;
                        ref = sk;
                    } else if (sk != -INFINITY) {
                        L += ex2(sk - ref);
                    }
                }
                fo = L != 0.f ? __fdividef(fo, L) : 0.f;
                uint16_t* y = (uint16_t*)a.out + (size_t)(cw.s.c0 + tok) * a.o_tok + hq * a.o_head + d;
                *reinterpret_cast<uint32_t*>(y) =
                    a.bf16 ? pack2<GRAFT_BF16>(x.x * fo, x.y * fo) : pack2<GRAFT_F16>(x.x * fo, x.y * fo);
                if (a.lse && d == 0)
                    a.lse[(size_t)(cw.s.c0 + tok) * a.q_heads + hq] = L != 0.f ? (ref + lg2(L)) * kLn2 : -INFINITY;
            };
            int ca, cb;
            split.cuts(cw.p0, cw.p0 + cw.nu, ca, cb);
            if (cb < ca) {
#pragma unroll 1
                for (int r = r0; r < R; r += STEP)
                    finish(r, *reinterpret_cast<const float2*>(&sum[r * DP + d]), joined[r].x, joined[r].y);
            } else {   // pieces of the pair meet in the workspace; its last CTA adds them up
                const int firstc = ca - 1, pieces = cb - ca + 2;
                float* slot = a.partials + ((size_t)blockIdx.x * 2 + (cw.lo == cw.u0)) * C::PARTIAL;
#pragma unroll 1
                for (int r = r0; r < R; r += STEP)
                    __stcg(reinterpret_cast<float2*>(slot + r * DP + d), *reinterpret_cast<const float2*>(&sum[r * DP + d]));
                if (tid < R) __stcg(reinterpret_cast<float2*>(slot + N * DP) + tid, make_float2(joined[tid].x, joined[tid].y));
                both_sync();
                if (tid == 0) {
                    // (release: the CTA's partial result before its count; acquire: the others')
                    unsigned was;
                    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;"
                                 : "=r"(was) : "l"(a.counters + firstc) : "memory");
                    sh_last = was + 1 == (unsigned)pieces;
                    if (sh_last) a.counters[firstc] = 0;
                }
                both_sync();
                if (sh_last) {
                    const float* parts = a.partials + (size_t)firstc * 2 * C::PARTIAL;   // piece k: CTA firstc + k
#pragma unroll 1
                    for (int r = r0; r < R; r += STEP) {
                        float M = kNoMax, L = 0.f;
                        float2 x = make_float2(0.f, 0.f);
                        constexpr int KB = 8;   // pieces read at a time
#pragma unroll 1
                        for (int k0 = 0; k0 < pieces; k0 += KB) {
                            float2 ml[KB], v[KB];
#pragma unroll
                            for (int k = 0; k < KB; ++k) {
                                const int kk = min(k0 + k, pieces - 1);
                                const float* p = parts + (size_t)(2 * kk + (kk == 0)) * C::PARTIAL;
                                ml[k] = __ldcg(reinterpret_cast<const float2*>(p + N * DP) + r);
                                v[k] = __ldcg(reinterpret_cast<const float2*>(p + r * DP + d));
                            }
                            const float was = M;
#pragma unroll
                            for (int k = 0; k < KB; ++k) M = fmaxf(M, ml[k].x);
                            const float f0 = ex2(was - M);
                            L *= f0, x.x *= f0, x.y *= f0;
#pragma unroll
                            for (int k = 0; k < KB; ++k) {
                                const float fk = k0 + k < pieces ? ex2(ml[k].x - M) : 0.f;
                                L = fmaf(ml[k].y, fk, L), x.x = fmaf(v[k].x, fk, x.x), x.y = fmaf(v[k].y, fk, x.y);
                            }
                        }
                        finish(r, x, M, L);
                    }
                }
            }
            both_sync();   // (all that is shared has been read)
            if constexpr (TURNS) {   // the weights' buffers again: columns without a row to 0
                for (int i = tid; i < C::GROUPS * C::P_BYTES / 16; i += 32 * C::SOFT)
                    reinterpret_cast<uint4*>(sp)[i] = make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
                both_sync();
            }
        }
    } else if (warp < C::SOFT + C::CONV) {
        // ======================================================== converters
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        // A thread takes one chunk of 16 dims of every PER-th key: eight neighbours store to all banks (two
        // keys' four chunks of 64 dims).
        constexpr int PER = 64 / (DP / 16), NC = KT / PER;   // keys of a step; steps
        const int wl = (warp - C::SOFT) & 1;
        const bool of_v = warp - C::SOFT >= 2;
        const int chunk = DP == 64 ? lane & 3 : (lane & 3) | (lane >> 1 & 4);
        const int kr = DP == 64 ? wl * 8 + (lane >> 2) : wl * 4 + ((lane >> 2 & 1) | (lane >> 3 & 2));
        const bool dims = 16 * chunk < D;
        const uint8_t* mine = raw + of_v * C::CODES + kr * D + (dims ? 16 * chunk : 0);
        uint8_t* stages = (of_v ? sv : sk) + (chunk >> 2) * KT * 128 + kr * 128;
        uint64_t *full = of_v ? vfull : kfull, *freed = of_v ? vfree : kfree;
        for (int it = 0, slot = 0, lap = 0; next_piece(cw);) {
            const int begin = first_key(a, cw.s.start) & ~15, end = cw.s.start + cw.s.n;
            for (int u = cw.lo; u < cw.hi; ++u, ++it) {
                const int st = it % ST, round = it / ST;
                wait(&rawfull[slot], lap);
                if (!of_v && wl == 0) {
                    // (the slot's last unit is long done: its scores were begun before those of the unit
                    // whose stage is waited for in the last turn)
                    if (lane < KT / 16) {
                        const float vs = fmaxf(raw_scales[slot][1][lane], kKVScaleFloor), lv = lg2(vs);
                        scales[it % SC][lane] = make_float4(raw_scales[slot][0][lane], lv, ex2(-lv), 0.f);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&scfull[it % SC]));
                }
                if (round) wait(&freed[st], round - 1);
                const uint8_t* from = mine + slot * 2 * C::CODES;
                // (what no key of the sequence wrote may be anything: 0)
                const bool whole = u * KT >= begin && (u + 1) * KT <= end && dims;
                // (eight loads, then their stores: the compiler keeps a load behind a store to shared memory)
#pragma unroll
                for (int b = 0; b < NC; b += 8) {
                    uint4 x[8];
#pragma unroll
                    for (int c = 0; c < 8; ++c) x[c] = *reinterpret_cast<const uint4*>(from + (b + c) * PER * D);
                    if (!whole)
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            const int key = u * KT + (b + c) * PER + kr;
                            if (!(dims && key >= begin && key < end)) x[c] = make_uint4(0, 0, 0, 0);
                        }
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        uint8_t* line = stages + st * C::KV_BYTES + (b + c) * PER * 128;   // 16 dims: chunks 2 (chunk & 3), + 1
                        const int turn = ((b + c) * PER + kr) & 7;
                        uint32_t o[8];
                        codes_h2<FMT>(x[c].x, o[0], o[1]);
                        codes_h2<FMT>(x[c].y, o[2], o[3]);
                        codes_h2<FMT>(x[c].z, o[4], o[5]);
                        codes_h2<FMT>(x[c].w, o[6], o[7]);
                        *reinterpret_cast<uint4*>(line + (((2 * (chunk & 3)) ^ turn) << 4)) =
                            make_uint4(o[0], o[1], o[2], o[3]);
                        *reinterpret_cast<uint4*>(line + (((2 * (chunk & 3) + 1) ^ turn) << 4)) =
                            make_uint4(o[4], o[5], o[6], o[7]);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&full[st])), mbar_arrive(smem_u32(&rawfree[slot]));
                if (++slot == C::RAW) slot = 0, ++lap;
            }
        }
    } else if (warp == C::SOFT + C::CONV + 1) {
        // ============================================================ loader
        // Lane i < 8 copies the codes of keys 16 i .. of a unit (16 keys lie in one block); lanes 0-7 copy
        // the scales of K, 8-15 those of V.
        Walk w = cw;
        w.hi = 0;
        int u = 0, blk = 0;
        bool more = true;
        auto inside = [&](int key) { return (key | 15) >= first_key(a, w.s.start) && key < w.s.start + w.s.n; };
        auto lookup = [&]() {   // the next unit, and its blocks' numbers
            if (more && ++u >= w.hi) {
                more = next_piece(w);
                u = w.lo;
            }
            if (!more) return;
            const int key = u * KT + 16 * (lane & 7);
            blk = inside(key) ? a.table[(size_t)w.b * a.table_stride + (key >> a.bt_log2)] : -1;
        };
        lookup();
        int it = 0;
        for (; more; ++it) {
            const int slot = it % C::RAW, lap = it / C::RAW, key = u * KT + 16 * (lane & 7);
            const bool in = lane < 16 && inside(key);
            if (in && (uint32_t)blk >= a.n_blocks) {
                atomicOr(err, (unsigned)GRAFT_KV_EBLOCK);
                blk = 0;
            }
            const size_t bh = in ? (size_t)blk * H + w.h : 0;
            const size_t off = ((bh << a.bt_log2) + (key & ((1 << a.bt_log2) - 1))) * D;
            const uint32_t bar = smem_u32(&rawfull[slot]), bytes = 16 * D;
            const int copies = __popc(__ballot_sync(~0u, in && lane < 8));
            if (lap) wait(&rawfree[slot], lap - 1);
            __syncwarp();
            if (lane == 0) mbar_arrive_expect_tx(bar, 2 * copies * bytes);
            __syncwarp();
            if (in && lane < 8) {
                const uint32_t to = smem_u32(raw + slot * 2 * C::CODES) + lane * bytes;
                bulk_g2s(to, a.k + off, bytes, bar);
                bulk_g2s(to + C::CODES, a.v + off, bytes, bar);
            }
            if (lane < 16) {
                const float* from = (lane < 8 ? a.k_scale : a.v_scale) + bh;
                cp_async4_or_zero(smem_u32(&raw_scales[slot][lane >> 3][lane & 7]), from, in);
                cp_async_mbar_arrive(bar);
            }
            lookup();
        }
        // no copy is on its way when the CTA ends, also after a wait gave up
        for (int i = max(0, it - C::RAW); i < it; ++i) {
            uint64_t t0 = 0;
            while (!mbar_try_wait(smem_u32(&rawfull[i % C::RAW]), i / C::RAW & 1)) {
                const uint64_t now = global_ns();
                if (t0 == 0) t0 = now;
                if (now - t0 > kAttnWaitNs) {
                    atomicOr(err, (unsigned)GRAFT_KV_EWAIT);
                    break;
                }
            }
        }
    } else {
        // =============================================================== MMA
        // (the whole warp walks and waits; one lane issues)
        constexpr uint32_t iqk = tc5_idesc(N, false), ipv = tc5_idesc(N, true) | 1u << 15;   // (bit 15: A is M-major)
        const bool leader = elect_one();
        const uint32_t q0 = tc5_low(smem_u32(sq), 16), k0 = tc5_low(smem_u32(sk), 16);
        const uint32_t v0 = tc5_low(smem_u32(sv), KT * 128), p0 = tc5_low(smem_u32(sp), KT * 128);
        auto scores = [&](int it) {   // S^T = K q^T of unit it
            const int st = it % ST;
            spin(&kfull[st], it / ST);
            tc5_fence_after();
            if (leader) {
#pragma unroll
                for (int s = 0; s < DP / 16; ++s)
                    tc5_mma_ss(tmem + (it & 3) * N,
                               k0 + (st * C::KV_BYTES + (s / 4) * KT * 128 + (s & 3) * 32) / 16,
                               q0 + ((s / 4) * N * 128 + (s & 3) * 32) / 16, iqk, s > 0);
                tc5_commit(smem_u32(&sfull[it & 3]));
                tc5_commit(smem_u32(&kfree[st]));
            }
        };
        int done_units = 0, pc = 0;
        while (next_piece(cw)) {
            const int n = cw.hi - cw.lo;
            spin(&qfull, pc);
            for (int j = 0; j < C::AHEAD && j < n; ++j) scores(done_units + j);
            for (int j = 0; j < n; ++j) {
                const int it = done_units + j, st = it % ST, b = it & 1;
                spin(&pfull[b], it >> 1);
                spin(&vfull[st], it / ST);
                tc5_fence_after();
                if (leader) {   // O^T += V^T P
#pragma unroll
                    for (int s = 0; s < KT / 16; ++s)
                        tc5_mma_ss(tmem + C::O_COL + (TURNS ? b * N : 0), v0 + (st * C::KV_BYTES + s * 2048) / 16,
                                   p0 + (b * C::P_BYTES + s * 2048) / 16, ipv, j > (TURNS ? 1 : 0) || s > 0);
                    tc5_commit(smem_u32(&pdone[b]));
                    tc5_commit(smem_u32(&vfree[st]));
                }
                // (the weights' arrival says that their scores have been read)
                if (j + C::AHEAD < n) scores(it + C::AHEAD);
            }
            done_units += n;
            ++pc;
        }
        if (leader) tc5_commit(smem_u32(&done));   // arrives once every product has completed
    }
    __syncthreads();
    if (warp == C::SOFT + C::CONV) {
        uint64_t t0 = 0;   // (bounded like the other waits, also after one of them gave up)
        while (!mbar_try_wait(smem_u32(&done), 0)) {
            const uint64_t now = global_ns();
            if (t0 == 0) t0 = now;
            if (now - t0 > kAttnWaitNs) {
                atomicOr(err, (unsigned)GRAFT_KV_EWAIT);
                break;
            }
        }
        __syncwarp();
        tc5_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512)
                     : "memory");
    }
}

}  // namespace dev
}  // namespace graft
