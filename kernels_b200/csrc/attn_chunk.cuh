// attn_chunk.cuh -- attention over the 8-bit cache for many query rows a head
// (chunks of a prompt), on the fifth-generation tensor cores.
//
// Rows are (token, query head of the key/value head) pairs.  A CTA (one per SM)
// works on RT tiles of 128 rows against units of KT keys, with O and the scores
// in tensor memory and these roles:
//   softmax     (4 warps a row tile)  thread = row = TMEM lane: reads its KT scores,
//               takes the weights and writes them back as fp16 (the A operand
//               of the second product) over the scores;
//   converters  (4 warps)  read a unit's codes from the cache and store them as
//               fp16 in shared memory, 128-byte swizzled rows of 64 dims: the
//               K-major B operand of q K^T and, unchanged in layout, the
//               MN-major B operand of P V;
//   MMA         (one lane)  per row tile and half unit of 64 keys: q K^T of half
//               j + 2 and P V of half j.
// Scores and weights are double-buffered by the half's parity, so a tile's softmax
// finds the next half's scores ready when it ends one: its chain is not
// lengthened by the products.
// The scales enter the exponents as in the few-row kernel (attn_few.cuh).  The
// reference of the exponents follows the row's maximum only when it is passed by
// more than kPSlack, so that O is seldom rescaled in tensor memory.
// Work is split evenly over the CTAs by (row tile, head, unit), and the pieces of
// a cut pair meet in the workspace (Split in attn_common.cuh).
//
// What bounds it: the softmax warps.  Chunks of 1024, 777 and 57 tokens behind 1024 to
// 4001 cached ones, 64 query heads on 8 of 64: 172 us, 423 TFLOP/s; 2048 last tokens of
// 5120: issue 39%, tensor pipe 23% (281 us cold).  An SM ends a half of 64 keys every 1400 cycles
// (at 1.9 GHz), so each of its two tiles' warps take about 2800 for one: a chain of waiting,
// loading, exponentials and storing, in which the exponentials of both tiles keep the MUFU busy
// for 1024.  When the call took 169 us, it took 143 without the exponentials, 119 without any
// softmax, 170 without the conversion and 175 without P V.
#pragma once
#include "attn_common.cuh"

#include <type_traits>

namespace graft {
namespace dev {

template <int DP>
struct Chunk {
    static constexpr int RT = DP <= 128 ? 2 : 1;     // row tiles
    static constexpr int KT = DP <= 128 ? 128 : 64;  // keys of a unit (one stage of K and V)
    static constexpr int HN = KT / 64;               // its halves of 64 keys (one product each)
    static constexpr int ST = DP <= 64 ? 3 : 2;      // stages
    static constexpr int ROWS = 128 * RT;
    static constexpr int SOFT = 4 * RT;              // softmax warps
    static constexpr int THREADS = 32 * (SOFT + 4 + 1);
    static constexpr int DB = DP / 64;               // blocks of 64 dims
    static constexpr int Q_BYTES = RT * DB * 128 * 128;
    static constexpr int KV_BYTES = DB * KT * 128;   // K or V of a unit
    static constexpr int SMEM = 1024 + Q_BYTES + 2 * ST * KV_BYTES;
    // TMEM columns: scores of tile i, half of parity b at i*128 + b*64; its weights (two fp16 a
    // column) over the scores, or where there is room beside them; its output.
    static constexpr bool BESIDE = DP != 128;
    static constexpr int P_COL = DP <= 64 ? 256 : DP <= 128 ? 0 : 128;
    static constexpr int P_TILE = DP <= 64 ? 64 : 128, P_STEP = DP == 128 ? 64 : 32;
    static constexpr int O_COL = DP <= 64 ? 384 : 256;
    // Weights are 2^(t - m), the reference m SHIFT below the largest t that it was taken
    // from.  Where a half is weighed before its maximum is known, fp16 leaves room for scores
    // up to 12 (in log2) above that, and keeps its 11 bits down to 17 below it (nothing is left
    // 28 below); the reference goes up only near that limit, because O's rescaling waits for
    // the product before.  (Shifts of 5 and 8, which keep more, make it go up more often:
    // the chunks above 177 and 187 us, 172 with 3.)
    static constexpr float SHIFT = BESIDE ? 3.f : kPShift;
    static constexpr int SC = 8;                     // slots of a unit's scales (up to ST + 2 in use)
    // floats of a partial result: O column by column, reference and sum of each row
    static constexpr int PARTIAL = ROWS * DP + 2 * ROWS;
};

// ---- tcgen05 (inline PTX)
__device__ __forceinline__ void tc5_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc5_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc5_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                     bar)
                 : "memory");
}
// D (+)= A B: A from shared memory or from tensor memory, B from shared memory.
// Descriptors of 128-byte swizzled rows as two words: low, start address >> 4 and
// leading byte offset >> 4; high, the constant part (stride byte offset 1024 >> 4,
// version 1, SWIZZLE_128B).  K-major: groups of 8 rows are 1024 bytes apart.
// MN-major: groups of 8 along K are 1024 bytes, blocks of 64 along MN `lead` apart.
constexpr uint32_t kTc5High = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t tc5_low(uint32_t addr, uint32_t lead) {
    return (addr >> 4) | ((lead >> 4) << 16);
}
__device__ __forceinline__ void tc5_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                           uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kTc5High)
        : "memory");
}
__device__ __forceinline__ void tc5_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                           uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kTc5High)
        : "memory");
}
// One lane of a converged warp, always the same.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(p));
    return p != 0;
}
// kind::f16 instruction descriptor: f32 sums, fp16 operands, M = 128, N; bit 16: B is MN-major.
__device__ __forceinline__ constexpr uint32_t tc5_idesc(int n, bool mn_major) {
    return (1u << 4) | (mn_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
        "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
        "%30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
          "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
          "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]),
          "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]),
          "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
        "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, "
        "%29, %30, %31, %32};" ::"r"(addr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
        "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]),
        "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
        "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

template <int DP, int FMT>
__global__ void __launch_bounds__(Chunk<DP>::THREADS, 1)
    attn_chunk_kernel(const __grid_constant__ AttnArgs a, unsigned* err) {
    using C = Chunk<DP>;
    constexpr int RT = C::RT, KT = C::KT, ST = C::ST, SC = C::SC, DB = C::DB, ROWS = C::ROWS;
    struct Walk {
        long long at, prefix;   // next key; keys (with the pads, of all heads) before the row tile
        long long p0;           // first key of the pair
        Seq s;
        int b, rt, tiles;       // sequence, row tile, row tiles of the sequence
        int nk, k0, k1;         // keys of the row tile a head with the pad; first key, last + 1
        int h, lo, hi;          // the piece: head, units [lo, hi)
    };
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Walk sh_edge[2];
    __shared__ uint64_t kfull[ST], kfree[ST], vfull[ST], vfree[ST], scfull[SC], qfull[RT], done;
    __shared__ uint64_t sfull[RT][2], pfull[RT][2], pdone[RT][2];   // by the half's parity
    __shared__ float4 scales[SC][KT / 16];   // k_scale, log2(v_scale), 1 / v_scale
    __shared__ uint32_t tmem_at;
    __shared__ volatile int dead;            // a wait gave up: every role stops
    __shared__ long long sh_scan[C::THREADS / 32];
    __shared__ int sh_last[RT];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int D = a.dim, H = a.heads, G = a.group, TT = ROWS / G;   // tokens of a row tile
    uint8_t* base = smem + ((1024 - (smem_u32(smem) & 1023)) & 1023);
    uint8_t *sq = base, *sk = base + C::Q_BYTES, *sv = sk + ST * C::KV_BYTES;
    if (tid == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(smem_u32(&kfull[i]), 4), mbar_init(smem_u32(&vfull[i]), 4);   // converter warps
            mbar_init(smem_u32(&kfree[i]), 1), mbar_init(smem_u32(&vfree[i]), 1);   // commits
        }
        for (int i = 0; i < SC; ++i) mbar_init(smem_u32(&scfull[i]), 4);
        for (int i = 0; i < RT; ++i) {
            mbar_init(smem_u32(&qfull[i]), 4);             // softmax warps
            for (int b = 0; b < 2; ++b) {
                mbar_init(smem_u32(&pfull[i][b]), 4);
                mbar_init(smem_u32(&sfull[i][b]), 1), mbar_init(smem_u32(&pdone[i][b]), 1);   // commits
            }
        }
        mbar_init(smem_u32(&done), 1);
        dead = 0;
    }
    fence_mbar_init();
    pdl_wait();
    pdl_launch_dependents();

    // ---- keys of a row tile and of the row tiles before it
    auto open_tile = [&](Walk& w) {
        const int i0 = w.rt * TT, i1 = min(w.s.n, i0 + TT);
        w.k0 = first_key(a, w.s.start + i0), w.k1 = w.s.start + i1;
        w.nk = w.k1 - w.k0 + a.pad_units;
    };
    auto open_seq = [&](Walk& w) {
        w.s = load_seq(a, w.b, err);
        w.tiles = (w.s.n + TT - 1) / TT;
    };
    auto keys_before = [&](const Walk& w, int rt) {   // rt <= tiles
        return tile_keys(w.s.start, w.s.n, TT, w.tiles, rt, (int)a.window, a.pad_units);
    };
    Split<long long> sp;
    Walk cw;
    long long fe;
    {
        long long U = 0, prefix = 0, base = 0;
        int pairs = 0;
        auto scan = [&](long long v, long long& before) {   // over the CTA's threads; the total
            long long x = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(~0u, x, o);
                if (lane >= o) x += y;
            }
            __syncthreads();
            if (lane == 31) sh_scan[warp] = x;
            __syncthreads();
            before = x - v;
            long long total = 0;
            for (int w = 0; w < C::THREADS / 32; ++w) {
                const long long y = sh_scan[w];
                if (w < warp) before += y;
                total += y;
            }
            return total;
        };
        long long mine = 0;
        for (uint32_t b0 = 0; b0 < a.n_seqs; b0 += C::THREADS) {
            cw.b = b0 + tid, cw.tiles = 0;
            if (cw.b < (int)a.n_seqs) open_seq(cw);
            mine = cw.tiles ? keys_before(cw, cw.tiles) : 0;
            U += scan(mine, prefix);
            pairs += __reduce_add_sync(~0u, cw.tiles);   // (this warp's; summed below)
        }
        if (U == 0) return;
        {
            long long skip;
            pairs = (int)scan(lane == 0 ? pairs : 0, skip) * H;
        }
        U *= H;
        const int grid = (int)min((long long)gridDim.x,
                                  max((long long)pairs, (U - (long long)pairs * a.pad_units) /
                                                            (a.min_units * KT)));
        if ((int)blockIdx.x >= grid) return;
        sp.set(U, grid, a.pad_units, a.min_units / 2 * KT);
        const long long x0 = sp.bound(blockIdx.x), x1 = sp.bound(blockIdx.x + 1);
        for (uint32_t b0 = 0; b0 < a.n_seqs; b0 += C::THREADS) {   // the bounds' sequences
            if (a.n_seqs > C::THREADS) {   // (else all is still at hand)
                cw.b = b0 + tid, cw.tiles = 0;
                if (cw.b < (int)a.n_seqs) open_seq(cw);
                mine = cw.tiles ? keys_before(cw, cw.tiles) : 0;
                const long long total = scan(mine, prefix);
                prefix += base;
                base += total;
            }
            cw.prefix = prefix * H;
            const long long e = cw.prefix + mine * H;
            if (cw.prefix <= x0 && x0 < e) sh_edge[0] = cw;
            if (cw.prefix <= x1 && x1 < e) sh_edge[1] = cw;
        }
        __syncthreads();
        // their row tiles: the CTA's threads test every step-th row tile, then the ones between
        auto find_tile = [&](int k, long long x) {
            Walk w = sh_edge[k];
            const long long seq_at = w.prefix;
            int lo = 0, n = w.tiles;   // the row tile is one of [lo, lo + n)
            while (n > 0) {
                const int step = (n + C::THREADS - 1) / C::THREADS, rt = lo + tid * step;
                __syncthreads();
                if (tid * step < n) {
                    const int end = min(rt + step, lo + n);
                    const long long p = seq_at + keys_before(w, rt) * H;
                    if (p <= x && x < seq_at + keys_before(w, end) * H) {
                        w.rt = rt;
                        w.prefix = p;
                        sh_edge[k] = w;
                    }
                }
                __syncthreads();
                if (step == 1) break;
                const int end = lo + n;
                lo = sh_edge[k].rt;
                n = min(step, end - lo);
            }
            w = sh_edge[k];
            open_tile(w);
            return w;
        };
        auto edge = [&](const Walk& w, long long x) {
            const long long p0 = w.prefix + (int)(x - w.prefix) / w.nk * w.nk;
            return sp.snapped(x, p0, p0 + w.nk);
        };
        fe = U;
        if (x1 < U) fe = edge(find_tile(1, x1), x1);
        cw = find_tile(0, x0);
        cw.at = edge(cw, x0);
        if (cw.at >= fe) return;
    }
    auto next_piece = [&](Walk& w) {   // false: no more
        if (w.at >= fe) return false;
        while (w.at >= w.prefix + (long long)w.nk * H) {
            w.prefix += (long long)w.nk * H;
            if (++w.rt >= w.tiles) {
                w.rt = 0;
                do {
                    ++w.b;
                    open_seq(w);
                } while (w.tiles == 0);
            }
            open_tile(w);
        }
        w.h = (int)(w.at - w.prefix) / w.nk;
        w.p0 = w.prefix + (long long)w.h * w.nk;
        const int from = (int)(w.at - w.p0), to = (int)(min(fe, w.p0 + w.nk) - w.p0);
        w.lo = (w.k0 + max(0, from - a.pad_units)) / KT;
        w.hi = to == w.nk ? (w.k1 - 1) / KT + 1 : (w.k0 + to - a.pad_units) / KT;
        w.at = w.p0 + to;
        return true;
    };
    // A wait for a barrier's phase.  When it gives up it sets an error bit and `dead`, after
    // which no wait waits: every role runs through its (bounded) loops and the call ends with
    // undefined outputs.  The MMA warp, whose lateness all others feel, spins on probes that
    // do not suspend (a suspended one wakes up to half a microsecond late).
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
    if (warp == C::SOFT + 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&tmem_at)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc5_fence_before();
    __syncthreads();
    tc5_fence_after();
    const uint32_t tmem = tmem_at;

    if (warp < C::SOFT) {
        // =========================================================== softmax
        // (registers move from the converters: 8 x 152 + 4 x 80, or 8 x 136 + 4 x 112, = 12 x 128)
        if constexpr (DP <= 64) asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
        else if constexpr (DP <= 128) asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
        const int tile = warp >> 2, row = (warp & 3) * 32 + lane;   // row of the tile = TMEM lane
        const uint32_t tlane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t ts0 = tlane + tile * 128, tp0 = tlane + C::P_COL + tile * C::P_TILE;
        const uint32_t to = tlane + C::O_COL + tile * DP;
        int it = 0, hc = 0;   // units and halves done
        while (next_piece(cw)) {
            const int r = tile * 128 + row, tok = cw.rt * TT + r / G, hq = cw.h * G + r % G;
            const bool on = r < TT * G && tok < cw.s.n;
            // ---- the row's queries, as fp16 (the sign of the scale goes with them)
            float cr;
            {
                const uint16_t* src = (const uint16_t*)a.q + (size_t)(cw.s.c0 + (on ? tok : 0)) * a.q_tok +
                                      (size_t)(on ? hq : 0) * a.q_head;
                float down = 1.f, up = 1.f;
                if (a.bf16) {
                    float amax = 0.f;
                    for (int d = 0; d < D && on; d += 8) {
                        const uint4 x = *reinterpret_cast<const uint4*>(src + d);
                        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 p = unpack2<GRAFT_BF16>(w[e]);
                            amax = (p.x == p.x) ? fmaxf(amax, fabsf(p.x)) : INFINITY;
                            amax = (p.y == p.y) ? fmaxf(amax, fabsf(p.y)) : INFINITY;
                        }
                    }
                    const float e = bf16_row_exponent(amax);
                    down = exp2f(-e), up = exp2f(e);
                }
                const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
                cr = fabsf(a.scale) * kLog2e * up;
#pragma unroll
                for (int c0 = 0; c0 < DP / 8; c0 += 8) {   // eight loads in flight
                    uint4 x[8];
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        x[c] = make_uint4(0, 0, 0, 0);
                        if (on && 8 * (c0 + c) < D) x[c] = *reinterpret_cast<const uint4*>(src + 8 * (c0 + c));
                    }
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        uint32_t w[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (a.bf16) {
                                const float2 p = unpack2<GRAFT_BF16>(w[e]);
                                w[e] = pack_h2(p.x * down, p.y * down);
                            }
                            w[e] ^= flip;
                        }
                        *reinterpret_cast<uint4*>(sq + ((tile * DB + c0 / 8) * 128 + row) * 128 +
                                                  ((c ^ (row & 7)) << 4)) =
                            make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                fence_proxy_async_smem();
                tc5_fence_before();   // (the last piece's O has been read)
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&qfull[tile]));
            }
            // (rows without a token need no mask: nothing of theirs is kept)
            const int p = on ? cw.s.start + tok : 1 << 30, lo = on ? first_key(a, p) : 0;
            float m = kNoMax, l = 0.f;   // reference, sum of the weights
            int raise = 0;               // of the reference, before the next unit
            // A reference beyond 2^20 (of any row of the warp): what is below is then worked out
            // as rounded scores, whose differences are exact.  The shorter form's sum of a scale
            // and the reference would be off by whole steps, and 2^(t - m) beyond fp16.
            // (Rows without a key yet and infinite ones do not count.)
            bool wide = false, careful;   // (careful: a unit that needs masks, or exact differences)
            auto widen = [&]() {
                wide = __any_sync(~0u, fabsf(m) > 0x1p20f && m != kNoMax && m < INFINITY);
                careful |= wide;
            };
            for (int u = cw.lo; u < cw.hi; ++u, ++it) {
                const bool first_unit = u == cw.lo;
                const int c_lo = lo - u * KT, c_hi = p - u * KT;   // columns that the row sees
                careful = wide || __any_sync(~0u, c_lo > 0 || c_hi < KT - 1);
                wait(&scfull[it % SC], it / SC);
                float top = 0.f;
#pragma unroll
                for (int hh = 0; hh < C::HN; ++hh, ++hc) {   // its halves
                const int b = C::HN == 1 ? hc & 1 : hh;
                const uint32_t ts = ts0 + b * 64, tp = tp0 + b * C::P_STEP;
                const float4* sc = scales[it % SC] + hh * 4;
                wait(&sfull[tile][b], hc >> 1);
                tc5_fence_after();
                auto rescale = [&](float f) {   // O, once the half before has been added
                    wait(&pdone[tile][b ^ 1], (hc - 1) >> 1);
                    tc5_fence_after();
#pragma unroll 1
                    for (int c = 0; c < DP / 32; ++c) {
                        uint32_t v[32];
                        tmem_ld32(to + 32 * c, v);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
                        tmem_st32(to + 32 * c, v);
                    }
                    tmem_wait_st();   // (a second rescaling reads what this one stored)
                };
                // ---- the row's maximum leads the reference of the exponents
                auto follow = [&](auto masked) {
                    float mx = -INFINITY;
#pragma unroll 1
                    for (int c = 0; c < 2; ++c) {
                        uint32_t v[32];
                        tmem_ld32(ts + 32 * c, v);
                        tmem_wait_ld();
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const float4 f = sc[2 * c + q];
                            float x = -INFINITY;
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                float y = __uint_as_float(v[16 * q + e]);
                                const int col = 64 * hh + 32 * c + 16 * q + e;
                                if (decltype(masked)::value) y = col >= c_lo && col <= c_hi ? y : -INFINITY;
                                x = fmaxf(x, y);
                            }
                            x = x == -INFINITY ? x : fmaf(x, f.x * cr, f.y);
                            mx = fmaxf(mx, x);
                        }
                    }
                    if (!__any_sync(~0u, mx - m > C::SHIFT + (C::BESIDE ? 0.f : kPSlack))) return;
                    const float up = fmaxf(m, reference(mx, C::SHIFT)), f = ex2(m - up);
                    l *= f;
                    m = up;
                    widen();
                    if (!first_unit || hh) rescale(f);
                };
                // ---- the weights; the largest sum of 16 of them
                float dl;
                auto weigh = [&](auto masked) {   // (masked: with exact differences too)
                    // (all 64 scores at once: straight code that keeps the MUFU fed, two
                    // fp32 operations an instruction where there are such)
                    float most = 0.f;
                    dl = 0.f;
                    uint32_t v[64];
                    tmem_ld32(ts, reinterpret_cast<uint32_t(&)[32]>(v[0]));
                    tmem_ld32(ts + 32, reinterpret_cast<uint32_t(&)[32]>(v[32]));
                    tmem_wait_ld();
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float4 f = sc[c];
                        const float fa = f.x * cr, fb = decltype(masked)::value ? f.y : f.y - m;
                        const uint64_t fa2 = pair(fa, fa), fb2 = pair(fb, fb);
                        uint64_t sum = 0;
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            const int col = 16 * c + e;
                            float x, y;
                            const uint64_t t2 = fma2(pair(__uint_as_float(v[col]), __uint_as_float(v[col + 1])), fa2, fb2);
                            unpair(decltype(masked)::value ? add2(t2, pair(-m, -m)) : t2, x, y);
                            if (decltype(masked)::value) {
                                const int at = 64 * hh + col;
                                x = at >= c_lo && at <= c_hi ? x : -INFINITY;
                                y = at + 1 >= c_lo && at + 1 <= c_hi ? y : -INFINITY;
                            }
                            x = ex2(x), y = ex2(y);
                            sum = add2(sum, pair(x, y));
                            v[8 * c + e / 2] = pack_h2(x, y);
                        }
                        float s0, s1;
                        unpair(sum, s0, s1);
                        s0 += s1;
                        most = fmaxf(most, s0);
                        dl = fmaf(s0, f.z, dl);
                    }
                    tmem_st32(tp, reinterpret_cast<uint32_t(&)[32]>(v[0]));
                    return most;
                };
                // Where the weights lie beside the scores, a half is weighed with the reference
                // that the halves before left, and weighed again in the rare case that a row
                // reached fp16's limit (no weight reaches 2^15 unless a sum of 16 does).
                if (!C::BESIDE || (first_unit && hh == 0)) {
                    if (careful) follow(std::true_type{});
                    else follow(std::false_type{});
                } else if (hh == 0 && __any_sync(~0u, raise > 0)) {
                    // by a power of two: the rows' sums and O keep their bits
                    const float up = m + (float)raise, f = ex2(m - up);
                    l *= f;
                    m = up;
                    widen();
                    rescale(f);
                }
                // (Once: no score lies more than SHIFT above the reference that follows it.)
                float most;
                for (bool again = false;; again = true) {
                    most = careful ? weigh(std::true_type{}) : weigh(std::false_type{});
                    if (!C::BESIDE || again || !__any_sync(~0u, most > 32768.f)) break;
                    tmem_wait_st();   // (the weights are stored again where these lie)
                    if (careful) follow(std::true_type{});
                    else follow(std::false_type{});
                }
                top = fmaxf(top, most);
                l += dl;
                tmem_wait_st();
                tc5_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&pfull[tile][b]));
                }
                // the next unit's reference goes up once the weights come near the limit
                raise = C::BESIDE && top > 16384.f ? (int)(__float_as_uint(top) >> 23) - 127 - (int)C::SHIFT : 0;
            }
            wait(&pdone[tile][(hc - 1) & 1], (hc - 1) >> 1);
            tc5_fence_after();
            // ---- output: the row itself, or its part of a cut pair
            int ca, cb;
            sp.cuts(cw.p0, cw.p0 + cw.nk, ca, cb);
            const bool cut = cb >= ca;
            const int first = ca - 1, pieces = cb - ca + 2;
            if (cut) {
                float* part = a.partials + ((size_t)blockIdx.x * 2 + (cw.lo == cw.k0 / KT)) * C::PARTIAL + r;
#pragma unroll 1
                for (int c = 0; c < DP / 32; ++c) {
                    uint32_t v[32];
                    tmem_ld32(to + 32 * c, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        __stcg(part + (32 * c + e) * ROWS, __uint_as_float(v[e]));
                }
                __stcg(part + DP * ROWS, m);
                __stcg(part + DP * ROWS + ROWS, l);
                // the row tile's 4 warps; each row tile has its own count
                asm volatile("bar.sync %0, 128;" ::"r"(1 + tile) : "memory");
                if ((tid & 127) == 0) {
                    unsigned was;
                    unsigned* count = a.counters + first * RT + tile;
                    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;"
                                 : "=r"(was) : "l"(count) : "memory");
                    sh_last[tile] = was + 1 == (unsigned)pieces;
                    if (sh_last[tile]) *count = 0;
                }
                asm volatile("bar.sync %0, 128;" ::"r"(1 + tile) : "memory");
                if (!sh_last[tile]) continue;
            }
            const float* parts = a.partials + (size_t)first * 2 * C::PARTIAL + r;   // piece k: CTA first + k
            auto piece = [&](int k) { return parts + (size_t)(2 * k + (k == 0)) * C::PARTIAL; };
            if (cut) {
                m = kNoMax, l = 0.f;
                for (int k = 0; k < pieces; ++k) m = fmaxf(m, __ldcg(piece(k) + DP * ROWS));
                for (int k = 0; k < pieces; ++k)
                    l = fmaf(__ldcg(piece(k) + DP * ROWS + ROWS), ex2(__ldcg(piece(k) + DP * ROWS) - m), l);
            }
            float ref = m, fo = 1.f;
            if (a.sinks) {
                const float s = a.sinks[on ? hq : 0] * kLog2e;
                if (s > ref) {
                    fo = ex2(ref - s);
                    l = l * fo + 1.f;
                    ref = s;
                } else if (s != -INFINITY) {
                    l += ex2(s - ref);
                }
            }
            fo = l != 0.f ? __fdividef(fo, l) : 0.f;
            uint16_t* y = (uint16_t*)a.out + (size_t)(cw.s.c0 + (on ? tok : 0)) * a.o_tok +
                          (size_t)(on ? hq : 0) * a.o_head;
#pragma unroll 1
            for (int c = 0; c < DP / 32; ++c) {
                float o[32];
                if (!cut) {
                    tmem_ld32(to + 32 * c, reinterpret_cast<uint32_t(&)[32]>(o));
                    tmem_wait_ld();
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0.f;
                    for (int k = 0; k < pieces; ++k) {
                        const float* q = piece(k);
                        const float f = ex2(__ldcg(q + DP * ROWS) - m);
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = fmaf(__ldcg(q + (32 * c + e) * ROWS), f, o[e]);
                    }
                }
                if (!on) continue;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int d = 32 * c + 8 * k;
                    if (d >= D) break;
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x0 = o[8 * k + 2 * e] * fo, x1 = o[8 * k + 2 * e + 1] * fo;
                        w[e] = a.bf16 ? pack2<GRAFT_BF16>(x0, x1) : pack2<GRAFT_F16>(x0, x1);
                    }
                    *reinterpret_cast<uint4*>(y + d) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            if (a.lse && on)
                a.lse[(size_t)(cw.s.c0 + tok) * a.q_heads + hq] = l != 0.f ? (ref + lg2(l)) * kLn2 : -INFINITY;
        }
    } else if (warp < C::SOFT + 4) {
        // ======================================================== converters
        if constexpr (DP <= 64) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        else if constexpr (DP <= 128) asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
        constexpr int NC = DP * KT / (16 * 128);   // chunks of 16 codes of a thread, K and V each
        const int ct = tid - 32 * C::SOFT, row = ct % KT, c0 = ct / KT * NC;
        Walk w = cw;
        w.hi = 0;
        int u = 0, blk = 0;
        bool more = true;
        // Keys that a row of the tile sees, and those that share 16 with one: a block before the
        // window may be gone.  (16 keys lie in one block.)
        auto inside = [&](int key) { return (key | 15) >= w.k0 && key < w.s.start + w.s.n; };
        auto lookup = [&]() {   // the next unit, and the number of its key's block
            if (more && ++u >= w.hi) {
                more = next_piece(w);
                u = w.lo;
            }
            if (!more) return;
            const int key = u * KT + row;
            blk = inside(key) ? a.table[(size_t)w.b * a.table_stride + (key >> a.bt_log2)] : 0;
        };
        uint4 kc[NC], vc[NC];
        float ks = 0.f, vs = 1.f;
        auto fetch = [&]() {    // its codes, and the block's scales
            const int key = u * KT + row;
            const bool in = inside(key);
            if (in && (uint32_t)blk >= a.n_blocks) {
                atomicOr(err, (unsigned)GRAFT_KV_EBLOCK);
                blk = 0;
            }
            const size_t bh = (size_t)blk * H + w.h;
            const size_t off = ((bh << a.bt_log2) + (key & ((1 << a.bt_log2) - 1))) * D + 16 * c0;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const bool ok = in && 16 * (c0 + c) < D;
                kc[c] = ok ? ld_ro(a.k + off + 16 * c) : make_uint4(0, 0, 0, 0);
                vc[c] = ok ? ld_ro(a.v + off + 16 * c) : make_uint4(0, 0, 0, 0);
            }
            ks = in ? a.k_scale[bh] : 0.f;
            vs = in ? fmaxf(a.v_scale[bh], kKVScaleFloor) : 1.f;
        };
        auto store = [&](uint8_t* to, const uint4 (&x)[NC]) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int at = c0 + c;   // 16 dims: chunks 2 (at & 3), + 1 of a 128-byte row
                uint8_t* line = to + ((at >> 2) * KT + row) * 128;
                uint32_t o[8];
                codes_h2<FMT>(x[c].x, o[0], o[1]);
                codes_h2<FMT>(x[c].y, o[2], o[3]);
                codes_h2<FMT>(x[c].z, o[4], o[5]);
                codes_h2<FMT>(x[c].w, o[6], o[7]);
                *reinterpret_cast<uint4*>(line + (((2 * (at & 3)) ^ (row & 7)) << 4)) =
                    make_uint4(o[0], o[1], o[2], o[3]);
                *reinterpret_cast<uint4*>(line + (((2 * (at & 3) + 1) ^ (row & 7)) << 4)) =
                    make_uint4(o[4], o[5], o[6], o[7]);
            }
        };
        lookup();
        if (more) fetch();
        bool have = more;
        lookup();
        for (int it = 0; have; ++it) {
            const int st = it % ST, round = it / ST;
            if (round) wait(&kfree[st], round - 1);
            store(sk + st * C::KV_BYTES, kc);
            if (ct < KT && ct % 16 == 0) {   // (16 keys lie in one block)
                const float lv = lg2(vs);
                scales[it % SC][ct / 16] = make_float4(ks, lv, ex2(-lv), 0.f);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&kfull[st])), mbar_arrive(smem_u32(&scfull[it % SC]));
            if (round) wait(&vfree[st], round - 1);
            store(sv + st * C::KV_BYTES, vc);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&vfull[st]));
            have = more;
            if (more) fetch();
            lookup();
        }
    } else {
        // =============================================================== MMA
        // (the whole warp walks and waits; one lane issues)
        constexpr uint32_t iqk = tc5_idesc(64, false), ipv = tc5_idesc(DP, true);
        const bool leader = elect_one();
        const uint32_t q0 = tc5_low(smem_u32(sq), 16), k0 = tc5_low(smem_u32(sk), 16);
        const uint32_t v0 = tc5_low(smem_u32(sv), KT * 128);
        auto scores = [&](int tile, int hc) {   // S = q K^T of half hc
            const int st = hc / C::HN % ST;
            if (leader) {
#pragma unroll
                for (int s = 0; s < DP / 16; ++s)
                    tc5_mma_ss(tmem + tile * 128 + (hc & 1) * 64,
                               q0 + ((tile * DB + s / 4) * 128 * 128 + (s & 3) * 32) / 16,
                               k0 + (st * C::KV_BYTES + hc % C::HN * 64 * 128 +
                                     (s / 4) * KT * 128 + (s & 3) * 32) / 16, iqk, s > 0);
                tc5_commit(smem_u32(&sfull[tile][hc & 1]));
                if (tile == RT - 1 && hc % C::HN == C::HN - 1) tc5_commit(smem_u32(&kfree[st]));
            }
        };
        auto product = [&](int tile, int hc, bool accumulate) {   // O += P V
            const int st = hc / C::HN % ST;
            if (leader) {
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    tc5_mma_ts(tmem + C::O_COL + tile * DP,
                               tmem + C::P_COL + tile * C::P_TILE + (hc & 1) * C::P_STEP + 8 * s,
                               v0 + (st * C::KV_BYTES + hc % C::HN * 64 * 128 + s * 2048) / 16, ipv,
                               accumulate || s > 0);
                tc5_commit(smem_u32(&pdone[tile][hc & 1]));
                if (tile == RT - 1 && hc % C::HN == C::HN - 1) tc5_commit(smem_u32(&vfree[st]));
            }
        };
        auto wait_stage = [&](uint64_t* bars, int hc) {   // before a unit's first half
            if (hc % C::HN == 0) spin(&bars[hc / C::HN % ST], hc / C::HN / ST);
        };
        int hc = 0, pc = 0;
        while (next_piece(cw)) {
            const int n = (cw.hi - cw.lo) * C::HN;
            for (int j = 0; j < 2 && j < n; ++j) {   // the first two halves' scores
                wait_stage(kfull, hc + j);
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    if (j == 0) spin(&qfull[i], pc);
                    tc5_fence_after();
                    scores(i, hc + j);
                }
            }
            for (int j = 0; j < n; ++j, ++hc) {
                wait_stage(vfull, hc);
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    spin(&pfull[i][hc & 1], hc >> 1);
                    if (i == 0 && j + 2 < n) wait_stage(kfull, hc + 2);
                    tc5_fence_after();
                    // (in this order the scores' arrival says that the weights of the same
                    // parity have been read)
                    product(i, hc, j > 0);
                    if (j + 2 < n) scores(i, hc + 2);
                }
            }
            ++pc;
        }
        if (leader) tc5_commit(smem_u32(&done));   // arrives once every product has completed
    }
    __syncthreads();
    if (warp == C::SOFT + 4) {
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
