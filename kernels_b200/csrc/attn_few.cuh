// attn_few.cuh -- attention over the 8-bit cache for few query rows a head: up
// to 8*NT rows (tokens of a sequence x query heads of a key/value head), one
// pass over the keys.
//
// A warp works alone on units of UK keys: it keeps a ring of NS slots (K and V
// codes of a unit, as they lie in the cache) filled by bulk copies, decodes the
// codes to fp16 in registers and multiplies on the tensor cores with the *keys*
// (scores) and the *head's dims* (output) as the 16 rows of the MMA and the
// query rows as its 8 columns:
//   S^T [16 keys x 8 rows]  = K [16 x D] q^T [D x 8]
//   O^T [16 dims x 8 rows] += V^T [16 x 16 keys] P^T [16 keys x 8 rows]
// so that a group of 8 query heads wastes nothing, and the weights need only an
// 8 x 8 transpose (movmatrix) between the two products.  The order of the dims
// inside a product is free, so a lane loads 16 (K) or 8 (V) consecutive bytes.
//
// The scales: score = S (k_scale scale log2 e) is one factor per 16 keys.  The
// value's scale goes into the exponent: with t = score + log2(v_scale), the
// weight 2^(t - max t) times the bare code is the weighted value, and the sum
// of weights is that of 2^(t - max t) / v_scale, in fp32.
#pragma once
#include "attn_common.cuh"

namespace graft {
namespace dev {

constexpr int kFewWarps = 8;
constexpr int kFewThreads = 32 * kFewWarps;

template <int DP>
constexpr int kFewUnit = DP == 64 ? 32 : 16;   // keys of a unit
template <int DP, int NT>
constexpr bool kFewBig = NT * DP > 128;        // one CTA per SM (registers), a deeper ring
template <int DP, int NT>
constexpr int kFewRing = kFewBig<DP, NT> && DP != 256 ? 6 : 3;
template <int DP>
constexpr int kFewSlot = 2 * kFewUnit<DP> * DP + 32;   // K, V, scales of up to 2 blocks
constexpr int kFewMergeBytes = (kFewWarps / 2) * 16 * 32 * 4;
template <int DP, int NT>
constexpr int kFewSmem = kFewWarps * kFewRing<DP, NT> * kFewSlot<DP> + kFewMergeBytes;
// floats of a partial result: O, and the maximum and sum of each row
template <int DP, int NT>
constexpr int kFewPartial = (DP / 16) * NT * 4 * 32 + 2 * 8 * NT;

// The state of one warp: O^T and the running maximum and sum of its columns.
template <int DP, int NT>
struct FewState {
    float o[DP / 16][NT][4];
    float m[NT][2], l[NT][2];
    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int i = 0; i < DP / 16; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][n][e] = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = kNoMax, l[n][0] = l[n][1] = 0.f;
    }
};

template <int DP, int NT, int FMT>
__global__ void __launch_bounds__(kFewThreads, kFewBig<DP, NT> ? 1 : 2)
    attn_few_kernel(const __grid_constant__ AttnArgs a, unsigned* err) {
    constexpr int UK = kFewUnit<DP>, KT = UK / 16, NS = kFewRing<DP, NT>, W = kFewWarps;
    constexpr int ROWS = 8 * NT, CH = DP / 64;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint64_t bars[W * NS];
    __shared__ long long sh_scan[W + 1], sh_pairs[W + 1];
    __shared__ long long sh_prefix[2];
    __shared__ int sh_seq[2];
    __shared__ float sh_m[W][ROWS], sh_l[W][ROWS];
    __shared__ int sh_last;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int D = a.dim, H = a.heads;
    uint8_t* ring = smem + warp * NS * kFewSlot<DP>;
    float* merge = reinterpret_cast<float*>(smem + W * NS * kFewSlot<DP>);
    if (lane == 0)
        for (int i = 0; i < NS; ++i) mbar_init(smem_u32(&bars[warp * NS + i]), 33);
    fence_mbar_init();
    pdl_wait();
    pdl_launch_dependents();

    // ---- units of every sequence: their total, and where this CTA's bounds lie
    auto units_of = [&](const Seq& s, int& u0) {
        if (s.n == 0) return 0;
        u0 = first_key(a, s.start) / UK;
        return (s.start + s.n + UK - 1) / UK - u0;
    };
    auto scan_block = [&](long long v, long long* sh, long long& before, long long& total) {
        long long x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(~0u, x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) sh[warp] = x;
        __syncthreads();
        before = x - v, total = 0;
        for (int w = 0; w < W; ++w) {
            if (w < warp) before += sh[w];
            total += sh[w];
        }
    };
    Split sp;
    {
        long long U = 0, pairs = 0, before = 0;
        int mine = 0;   // units of sequence tid (kept for the usual case of up to 256 sequences)
        for (uint32_t b0 = 0; b0 < a.n_seqs; b0 += kFewThreads) {
            int u0, nu = 0;
            if (b0 + tid < a.n_seqs) nu = units_of(load_seq(a, b0 + tid, err), u0);
            long long bf, tot, pb, ptot;
            scan_block(nu, sh_scan, bf, tot);
            scan_block(nu > 0, sh_pairs, pb, ptot);
            if (b0 == 0) mine = nu, before = bf;
            U += tot, pairs += ptot;
        }
        U *= H, pairs *= H;
        if (U == 0) return;
        const long long want = (U + a.min_units - 1) / a.min_units;
        sp.U = U;
        sp.snap = max(1, a.min_units / 2);
        sp.G = (int)min((long long)gridDim.x, max(pairs, want));
        if ((int)blockIdx.x >= sp.G) return;
        const long long x0 = sp.bound(blockIdx.x), x1 = sp.bound(blockIdx.x + 1);
        if (tid == 0) sh_seq[1] = a.n_seqs, sh_prefix[1] = U;   // x1 = U: past the last
        __syncthreads();
        long long base = 0;
        for (uint32_t b0 = 0; b0 < a.n_seqs; b0 += kFewThreads) {
            int nu = mine;
            long long bf = before, tot = 0;
            if (a.n_seqs > kFewThreads) {
                int u0;
                nu = b0 + tid < a.n_seqs ? units_of(load_seq(a, b0 + tid, err), u0) : 0;
                scan_block(nu, sh_scan, bf, tot);
            }
            const long long p = (base + bf) * H, e = p + (long long)nu * H;
            if (p <= x0 && x0 < e) sh_seq[0] = b0 + tid, sh_prefix[0] = p;
            if (p <= x1 && x1 < e) sh_seq[1] = b0 + tid, sh_prefix[1] = p;
            base += tot;
        }
        __syncthreads();
    }
    // this CTA's units [f, fe)
    auto edge = [&](int i, long long x) {
        if (x >= sp.U) return sp.U;
        int u0;
        const int nu = units_of(load_seq(a, sh_seq[i], err), u0);
        const long long p0 = sh_prefix[i] + (x - sh_prefix[i]) / nu * nu;
        return sp.snapped(x, p0, p0 + nu);
    };
    long long f = edge(0, sp.bound(blockIdx.x));
    const long long fe = edge(1, sp.bound(blockIdx.x + 1));
    if (f >= fe) return;

    // A walk over the CTA's pieces of pairs.  Two run at a time: the one whose
    // units are being copied, and the one that is being computed.
    struct Walk {
        long long at, prefix;   // next unit, units before the sequence
        Seq s;
        int b, nu, u0;          // sequence, its units a head, its first unit
        int h, lo, hi;          // the piece: head, units [lo, hi) of the sequence
        long long p0;           // first unit of the pair
    };
    auto open_seq = [&](Walk& w) {
        w.u0 = 0;
        w.s = load_seq(a, w.b, err);
        w.nu = units_of(w.s, w.u0);
    };
    auto next_piece = [&](Walk& w) {   // false: no more
        if (w.at >= fe) return false;
        while (w.at >= w.prefix + (long long)w.nu * H) {
            w.prefix += (long long)w.nu * H;
            ++w.b;
            open_seq(w);
        }
        w.h = (int)((w.at - w.prefix) / w.nu);
        w.p0 = w.prefix + (long long)w.h * w.nu;
        const long long e = min(fe, w.p0 + w.nu);
        w.lo = w.u0 + (int)(w.at - w.p0);
        w.hi = w.u0 + (int)(e - w.p0);
        w.at = e;
        return true;
    };
    Walk cw;
    cw.b = sh_seq[0], cw.prefix = sh_prefix[0], cw.at = f;
    open_seq(cw);
    Walk iw = cw;

    // ---- copies: the next unit of this warp into ring slot `slot`
    bool more = next_piece(iw);
    int iu = more ? iw.lo + warp : 0;
    const int sub = min((int)a.bt, UK);   // tokens of a block in a unit
    auto issue = [&](int slot) {
        while (more && iu >= iw.hi) {
            more = next_piece(iw);
            iu = iw.lo + warp;
        }
        if (!more) return;
        const int key0 = iu * UK, valid = min(UK, iw.s.start + iw.s.n - key0);
        const uint32_t bar = smem_u32(&bars[warp * NS + slot]);
        uint8_t* sl = ring + slot * kFewSlot<DP>;
        const int n = (valid + sub - 1) / sub;
        int cnt = 0;
        size_t bh = 0;
        const int pos = key0 + lane * sub;
        if (lane < n) {
            const int blk = a.table[(size_t)iw.b * a.table_stride + pos / (int)a.bt];
            if ((uint32_t)blk < a.n_blocks) {
                bh = (size_t)blk * H + iw.h;
                cnt = min(sub, valid - lane * sub);
            } else {
                atomicOr(err, (unsigned)GRAFT_KV_EBLOCK);
            }
        }
        const int total = __reduce_add_sync(~0u, cnt);
        if (lane == 0) mbar_arrive_expect_tx(bar, 2 * total * D);
        __syncwarp();
        if (cnt > 0) {
            const size_t off = (bh * a.bt + pos % a.bt) * D;
            const uint32_t dst = smem_u32(sl) + lane * sub * D;
            bulk_g2s(dst, a.k + off, cnt * D, bar);
            bulk_g2s(dst + UK * DP, a.v + off, cnt * D, bar);
            const uint32_t sc = smem_u32(sl) + 2 * UK * DP + lane * 8;
            cp_async4(sc, a.k_scale + bh);
            cp_async4(sc + 4, a.v_scale + bh);
        }
        cp_async_mbar_arrive(bar);
        iu += W;
    };
#pragma unroll
    for (int i = 0; i < NS; ++i) issue(i);

    int q = 0;          // units this warp has taken from its ring
    bool dead = false;  // a wait gave up: nothing more is waited for
    FewState<DP, NT> st;
    uint32_t qf[CH][NT][8];
    float cn[NT][2];    // scale log2(e) of the columns' rows
    int pn[NT][2];      // positions of the columns' tokens

    // ---- joins the warps' states into warp 0's (every warp calls it)
    auto join = [&](int active) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c)
                if (g == 0) {
                    sh_m[warp][8 * n + 2 * t + c] = st.m[n][c];
                    sh_l[warp][8 * n + 2 * t + c] = st.l[n][c];
                }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int r = 8 * n + 2 * t + c;
                float M = kNoMax, L = 0.f;
                for (int w = 0; w < active; ++w) M = fmaxf(M, sh_m[w][r]);
                for (int w = 0; w < active; ++w) L += sh_l[w][r] * ex2(sh_m[w][r] - M);
                const float fct = ex2(st.m[n][c] - M);
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) st.o[i][n][c] *= fct, st.o[i][n][c + 2] *= fct;
                st.m[n][c] = M, st.l[n][c] = L;
            }
        // halves: 16 accumulators a lane at a time through shared memory
        for (int half = W / 2; half >= 1; half >>= 1) {
            if (active <= half) continue;
            constexpr int NO = (DP / 16) * NT * 4;
#pragma unroll
            for (int c0 = 0; c0 < NO; c0 += 16) {
                float* buf = merge + (warp & (half - 1)) * 16 * 32 + lane;
                if (warp >= half && warp < 2 * half && warp < active)
#pragma unroll
                    for (int e = 0; e < 16; ++e) buf[e * 32] = (&st.o[0][0][0])[c0 + e];
                __syncthreads();
                if (warp < half && warp + half < active)
#pragma unroll
                    for (int e = 0; e < 16; ++e) (&st.o[0][0][0])[c0 + e] += buf[e * 32];
                __syncthreads();
            }
            active = half;
        }
    };

    // ---- warp 0 writes a pair's finished rows
    auto finish = [&](const Walk& w) {
        const int R = w.s.n * (int)a.group;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int r = 8 * n + 2 * t + c;
                const bool on = r < R;
                const int tok = on ? r / (int)a.group : 0;
                const int hq = w.h * (int)a.group + (on ? r - tok * (int)a.group : 0);
                const float base = st.m[n][c] - kPShift;
                float L = st.l[n][c], fo = 1.f, ref = base;
                if (a.sinks) {
                    const float sk = a.sinks[hq] * kLog2e;
                    if (sk > base) {
                        fo = ex2(base - sk);
                        L = L * fo + 1.f;
                        ref = sk;
                    } else if (sk != -INFINITY) {
                        L += ex2(sk - base);
                    }
                }
                fo = L != 0.f ? __fdividef(fo, L) : 0.f;
                if (!on) continue;
                uint16_t* y = (uint16_t*)a.out + (size_t)(w.s.c0 + tok) * a.o_tok + hq * a.o_head;
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    const int d = 64 * i + 8 * g;
                    if (d >= D) break;
                    uint32_t v[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float x0 = st.o[4 * i + j][n][c] * fo, x1 = st.o[4 * i + j][n][c + 2] * fo;
                        v[j] = a.bf16 ? pack2<GRAFT_BF16>(x0, x1) : pack2<GRAFT_F16>(x0, x1);
                    }
                    *reinterpret_cast<uint4*>(y + d) = make_uint4(v[0], v[1], v[2], v[3]);
                }
                if (a.lse && g == 0)
                    a.lse[(size_t)(w.s.c0 + tok) * a.q_heads + hq] =
                        L != 0.f ? (ref + log2f(L)) * kLn2 : -INFINITY;
            }
    };

    while (next_piece(cw)) {
        const int R = cw.s.n * (int)a.group;
        st.reset();
        const bool has = cw.lo + warp < cw.hi;
        // ---- the pair's queries as B operands
        if (has) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int r = 8 * n + g;
                const bool on = r < R;
                const int tok = on ? r / (int)a.group : 0;
                const int hq = cw.h * (int)a.group + (on ? r - tok * (int)a.group : 0);
                const uint16_t* src = (const uint16_t*)a.q + (size_t)(cw.s.c0 + tok) * a.q_tok +
                                      hq * a.q_head;
                float amax = 0.f;
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    const int d = 64 * i + 16 * t;
                    uint4 x = make_uint4(0, 0, 0, 0), y = x;
                    if (on && d < D) {
                        x = *reinterpret_cast<const uint4*>(src + d);
                        y = *reinterpret_cast<const uint4*>(src + d + 8);
                    }
                    uint32_t* w = qf[i][n];
                    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
                    w[4] = y.x, w[5] = y.y, w[6] = y.z, w[7] = y.w;
                    if (a.bf16)
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float2 p = unpack2<GRAFT_BF16>(w[e]);
                            // (a NaN must not hide behind fmaxf)
                            amax = (p.x == p.x) ? fmaxf(amax, fabsf(p.x)) : INFINITY;
                            amax = (p.y == p.y) ? fmaxf(amax, fabsf(p.y)) : INFINITY;
                        }
                }
                float up = 1.f;
                if (a.bf16) {
                    amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
                    amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
                    const float e = bf16_row_exponent(amax), down = exp2f(-e);
                    up = exp2f(e);
#pragma unroll
                    for (int i = 0; i < CH; ++i)
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float2 p = unpack2<GRAFT_BF16>(qf[i][n][k]);
                            qf[i][n][k] = pack_h2(p.x * down, p.y * down);
                        }
                }
                const float c = a.scale * kLog2e * up;
                cn[n][0] = __shfl_sync(~0u, c, 8 * t);       // lane of row 2t (t = 0)
                cn[n][1] = __shfl_sync(~0u, c, 8 * t + 4);
#pragma unroll
                for (int c2 = 0; c2 < 2; ++c2)
                    pn[n][c2] = cw.s.start + min(8 * n + 2 * t + c2, R - 1) / (int)a.group;
            }
        }
        const int len = cw.s.start + cw.s.n;
        const int free_lo = first_key(a, len - 1);   // keys [free_lo, start] are seen by every row
        for (int u = cw.lo + warp; u < cw.hi; u += W, ++q) {
            const int slot = q % NS, key0 = u * UK;
            const uint32_t bar = smem_u32(&bars[warp * NS + slot]);
            uint8_t* sl = ring + slot * kFewSlot<DP>;
            if (!dead) {
                bool late = false;
                uint64_t t0 = 0;
                while (!late && !mbar_try_wait(bar, (q / NS) & 1)) {
                    const uint64_t now = global_ns();
                    if (t0 == 0) t0 = now;
                    late = now - t0 > kAttnWaitNs;
                }
                dead = __any_sync(~0u, late);
                if (dead && lane == 0) atomicOr(err, (unsigned)GRAFT_KV_EWAIT);
            }
            __syncwarp();
            const bool edge_unit = key0 < free_lo || key0 + UK - 1 > cw.s.start;
            const int valid = len - key0;   // (at least 1)
            const float* sc = reinterpret_cast<const float*>(sl + 2 * UK * DP);
            if (FMT == GRAFT_KV_E4M3 && valid < UK) {
                // what lies after the last token may be NaN codes: 0 * NaN is no weight
                uint8_t* vr = sl + UK * DP;
                for (int i = valid * D / 16 + lane; i < UK * D / 16; i += 32)
                    reinterpret_cast<uint4*>(vr)[i] = make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();   // (before a copy into this slot again)
                __syncwarp();
            }
            // ---- scores
            float s[KT][NT][4];
            float ivs[KT];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[kt][n][e] = 0.f;
                const uint8_t* kr = sl + (kt * 16 + g) * D + 16 * t;
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    uint4 x = make_uint4(0, 0, 0, 0), y = x;
                    if (64 * i + 16 * t < D) {
                        x = *reinterpret_cast<const uint4*>(kr + 64 * i);
                        y = *reinterpret_cast<const uint4*>(kr + 64 * i + 8 * D);
                    }
                    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t af[4];
                        codes_h2<FMT>(xs[k], af[0], af[2]);
                        codes_h2<FMT>(ys[k], af[1], af[3]);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            mma16816(s[kt][n], af, qf[i][n][2 * k], qf[i][n][2 * k + 1]);
                    }
                }
                // ---- t = score + log2(v_scale); the mask where the unit has one
                const int blk = kt * 16 / sub;
                const bool in = kt * 16 < valid;   // else no such block was copied
                const float ks = in ? sc[2 * blk] : 0.f;
                const float vs = in ? fmaxf(sc[2 * blk + 1], kKVScaleFloor) : 1.f;
                const float lv = log2f(vs);
                ivs[kt] = __fdividef(1.f, vs);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x = fmaf(s[kt][n][e], ks * cn[n][e & 1], lv);
                        if (edge_unit) {
                            const int j = key0 + kt * 16 + g + (e & 2) * 4, p = pn[n][e & 1];
                            const bool see = j <= p && (!a.window || j > p - (int)a.window);
                            x = see ? x : -INFINITY;
                        }
                        s[kt][n][e] = x;
                    }
            }
            // ---- running maximum, weights, their sum
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float mx[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float x = fmaxf(s[0][n][c], s[0][n][c + 2]);
#pragma unroll
                    for (int kt = 1; kt < KT; ++kt)
                        x = fmaxf(x, fmaxf(s[kt][n][c], s[kt][n][c + 2]));
                    x = fmaxf(x, __shfl_xor_sync(~0u, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(~0u, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(~0u, x, 16));
                    mx[c] = fmaxf(x, st.m[n][c]);
                }
                if (__any_sync(~0u, mx[0] > st.m[n][0] || mx[1] > st.m[n][1])) {
                    const float f0 = ex2(st.m[n][0] - mx[0]), f1 = ex2(st.m[n][1] - mx[1]);
                    st.l[n][0] *= f0, st.l[n][1] *= f1;
#pragma unroll
                    for (int i = 0; i < DP / 16; ++i) {
                        st.o[i][n][0] *= f0, st.o[i][n][2] *= f0;
                        st.o[i][n][1] *= f1, st.o[i][n][3] *= f1;
                    }
                    st.m[n][0] = mx[0], st.m[n][1] = mx[1];
                }
                const float b0 = st.m[n][0] - kPShift, b1 = st.m[n][1] - kPShift;
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    float* x = s[kt][n];
                    x[0] = ex2(x[0] - b0), x[1] = ex2(x[1] - b1);
                    x[2] = ex2(x[2] - b0), x[3] = ex2(x[3] - b1);
                    st.l[n][0] = fmaf(x[0] + x[2], ivs[kt], st.l[n][0]);
                    st.l[n][1] = fmaf(x[1] + x[3], ivs[kt], st.l[n][1]);
                }
            }
            // ---- O^T += V^T P^T
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                uint32_t pb[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    pb[n][0] = transpose8(pack_h2(s[kt][n][0], s[kt][n][1]));
                    pb[n][1] = transpose8(pack_h2(s[kt][n][2], s[kt][n][3]));
                }
                const uint8_t* vr = sl + UK * DP + (kt * 16 + 2 * t) * D + 8 * g;
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    uint2 w0 = make_uint2(0, 0), w1 = w0, w2 = w0, w3 = w0;
                    if (64 * i + 8 * g < D) {
                        w0 = *reinterpret_cast<const uint2*>(vr + 64 * i);
                        w1 = *reinterpret_cast<const uint2*>(vr + 64 * i + D);
                        w2 = *reinterpret_cast<const uint2*>(vr + 64 * i + 8 * D);
                        w3 = *reinterpret_cast<const uint2*>(vr + 64 * i + 9 * D);
                    }
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t A = x ? w0.y : w0.x, B = x ? w1.y : w1.x;
                        const uint32_t C = x ? w2.y : w2.x, E = x ? w3.y : w3.x;
                        uint32_t lo[4], hi[4];   // tiles 2x and 2x + 1
                        codes_h2<FMT>(prmt(A, B, 0x5140), lo[0], lo[1]);
                        codes_h2<FMT>(prmt(C, E, 0x5140), lo[2], lo[3]);
                        codes_h2<FMT>(prmt(A, B, 0x7362), hi[0], hi[1]);
                        codes_h2<FMT>(prmt(C, E, 0x7362), hi[2], hi[3]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma16816(st.o[4 * i + 2 * x][n], lo, pb[n][0], pb[n][1]);
                            mma16816(st.o[4 * i + 2 * x + 1][n], hi, pb[n][0], pb[n][1]);
                        }
                    }
                }
            }
            __syncwarp();
            issue(slot);
        }
        // ---- the lanes of a column hold sums over their own keys
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int o = 4; o < 32; o <<= 1)
                    st.l[n][c] += __shfl_xor_sync(~0u, st.l[n][c], o);
        join(min(W, cw.hi - cw.lo));

        // ---- a whole pair is finished; pieces meet in the workspace
        int ca, cb;
        sp.cuts(cw.p0, cw.p0 + cw.nu, ca, cb);
        if (cb < ca) {
            if (warp == 0) finish(cw);
            continue;
        }
        const int first = ca - 1, pieces = cb - ca + 2;
        constexpr int NO = (DP / 16) * NT * 4;
        const bool begins = cw.lo == cw.u0;   // this CTA holds the pair's first piece
        if (warp == 0) {
            float* p = a.partials + ((size_t)blockIdx.x * 2 + begins) * kFewPartial<DP, NT>;
#pragma unroll
            for (int e = 0; e < NO; ++e) __stcg(p + e * 32 + lane, (&st.o[0][0][0])[e]);
            p += NO * 32;
            if (g == 0)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        __stcg(p + 8 * n + 2 * t + c, st.m[n][c]);
                        __stcg(p + ROWS + 8 * n + 2 * t + c, st.l[n][c]);
                    }
            __threadfence();
            __syncwarp();
            if (lane == 0) {
                const unsigned was = atomicAdd(a.counters + first, 1u);
                sh_last = was + 1 == (unsigned)pieces;
                if (sh_last) a.counters[first] = 0;
            }
        }
        __syncthreads();
        if (!sh_last) continue;
        __threadfence();
        st.reset();
        for (int k = warp; k < pieces; k += W) {   // piece k: CTA first + k
            const float* p = a.partials + ((size_t)(first + k) * 2 + (k == 0)) * kFewPartial<DP, NT>;
            const float* ml = p + NO * 32;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float fo[2], fn[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float m2 = __ldcg(ml + 8 * n + 2 * t + c);
                    const float l2 = __ldcg(ml + ROWS + 8 * n + 2 * t + c);
                    const float M = fmaxf(st.m[n][c], m2);
                    fo[c] = ex2(st.m[n][c] - M), fn[c] = ex2(m2 - M);
                    st.l[n][c] = st.l[n][c] * fo[c] + l2 * fn[c];
                    st.m[n][c] = M;
                }
#pragma unroll
                for (int i = 0; i < DP / 16; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        st.o[i][n][e] = st.o[i][n][e] * fo[e & 1] +
                                        __ldcg(p + ((i * NT + n) * 4 + e) * 32 + lane) * fn[e & 1];
            }
        }
        join(min(W, pieces));
        if (warp == 0) finish(cw);
    }
}

}  // namespace dev
}  // namespace graft
