// attn_few.cuh -- attention over the 8-bit cache for few query rows a head: up
// to 8*NT rows (tokens of a sequence x query heads of a key/value head), one
// pass over the keys.
//
// A warp works alone on units of UK keys: it keeps a ring of NS slots (K and V
// codes of a unit, as they lie in the cache) filled by asynchronous copies
// (16 bytes a lane and instruction: with two addresses a unit they cost fewer
// instructions than a bulk copy with its barrier and byte count), decodes the
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
//
// What bounds it: HBM in long calls of wide heads (64 sequences of up to 8192 keys,
// 8 heads of 128, 4 query heads each, e4m3: 102 us, 5.3 TB/s; 32 of up to 8192, 8
// heads of 256: 101 us, 5.3 TB/s); with heads of 64 instruction issue as much (430 to
// 500 warp instructions a unit of 4 KB, 48% of the issue slots).  One sequence of 131071
// keys, 8 heads of 64, 64 query heads: 38.2 us, of which the stream is 21, the start (lengths,
// block numbers, first copies) 3.5 and the joins 7; where the other 7 go has not been found.
// Short calls are a chain of latencies: 517 keys 7.5 us, 32 sequences with a window of 128 and
// two tokens each 9.8 us.  17 to 32 rows take one CTA an SM (registers), whose 8 warps hide
// little: 32 sequences of up to 8192 keys 76 us, with 8 rows 41.
// Spills: instances for 16 rows of 64 dims 56 to 104 bytes, for 8 rows 28 to 40.
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
constexpr int kFewRing = kFewBig<DP, NT> && DP != 256 ? 4 : NT * DP > 64 ? 2 : 3;
template <int DP>
constexpr int kFewSlot = 2 * kFewUnit<DP> * DP + 16;   // K, V, scales of up to 2 blocks
template <int DP, int NT>
constexpr int kFewOut = (DP / 16) * NT * 4;    // accumulators of a lane
template <int DP, int NT>
constexpr int kFewSmem = kFewWarps * (kFewRing<DP, NT> * kFewSlot<DP> + kFewOut<DP, NT> * 32 * 4);
// floats of a partial result: O, and the reference and sum of each row
template <int DP, int NT>
constexpr int kFewPartial = kFewOut<DP, NT> * 32 + 2 * 8 * NT;

// The state of one warp: O^T and its columns' references and sums of weights.
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

template <int DP, int NT, int FMT, bool FULL>   // FULL: head_dim == DP
__global__ void __launch_bounds__(kFewThreads, kFewBig<DP, NT> ? 1 : 2)
    attn_few_kernel(const __grid_constant__ AttnArgs a, unsigned* err) {
    constexpr int UK = kFewUnit<DP>, KT = UK / 16, NS = kFewRing<DP, NT>, W = kFewWarps;
    constexpr int ROWS = 8 * NT, CH = DP / 64;
    constexpr int NB = UK / 16;   // most blocks that a unit touches
    // A walk over the CTA's pieces of pairs.  Two run at a time: the one whose
    // units are being copied, and the one that is being computed.
    struct Walk {
        int at, prefix;   // next unit, units before the sequence
        Seq s;
        int b, nu, u0;    // sequence, its units a head with the pad (0: none), its first unit
        int h, lo, hi;    // the piece: head, units [lo, hi) of the sequence
        int p0;           // first unit of the pair
    };
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Walk sh_edge[2];
    __shared__ int sh_scan[W];
    __shared__ float2 sh_ml[W][ROWS];
    __shared__ int sh_last;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int D = FULL ? DP : a.dim, H = a.heads;
    pdl_wait();
    pdl_launch_dependents();

    // ---- units of every sequence: their total, and where this CTA's bounds lie
    auto open_seq = [&](Walk& w) {
        w.s = load_seq(a, w.b, err);
        w.u0 = first_key(a, w.s.start) / UK;
        w.nu = w.s.n ? (w.s.start + w.s.n + UK - 1) / UK - w.u0 + a.pad_units : 0;
    };
    Split<int> sp;
    Walk cw;
    int fe;   // this CTA's units: [cw.at, fe)
    {
        int U = 0, pairs = 0, prefix = 0;
        // (the usual case of up to 256 sequences reads their lengths once)
        auto scan = [&](uint32_t b0, int base) {
            cw.b = b0 + tid, cw.nu = 0;
            if (cw.b < (int)a.n_seqs) open_seq(cw);
            int x = cw.nu;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(~0u, x, o);
                if (lane >= o) x += y;
            }
            if (lane == 31) sh_scan[warp] = x;
            pairs += __syncthreads_count(cw.nu > 0);
            prefix = base + x - cw.nu;
            int total = 0;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const int y = sh_scan[w];
                if (w < warp) prefix += y;
                total += y;
            }
            return total;
        };
        for (uint32_t b0 = 0; b0 < a.n_seqs; b0 += kFewThreads) {
            if (b0) __syncthreads();
            U += scan(b0, 0);
        }
        U *= H, pairs *= H;
        if (U == 0) return;
        // (more than pairs, while shares stay above a pad and a unit: few CTAs get two pairs)
        const int G = min((int)gridDim.x, max(max(pairs, (U - pairs * a.pad_units) / a.min_units),
                                              min(2 * pairs, U / (a.pad_units + 1))));
        if ((int)blockIdx.x >= G) return;
        sp.set(U, G, a.pad_units, a.min_units);
        const int x0 = sp.bound(blockIdx.x), x1 = sp.bound(blockIdx.x + 1);
        int base = 0;
        for (uint32_t b0 = 0; b0 < a.n_seqs; b0 += kFewThreads) {
            if (a.n_seqs > kFewThreads) {
                __syncthreads();
                base += scan(b0, base);
            }
            cw.prefix = prefix * H;
            const int e = cw.prefix + cw.nu * H;
            if (cw.prefix <= x0 && x0 < e) sh_edge[0] = cw;
            if (cw.prefix <= x1 && x1 < e) sh_edge[1] = cw;
        }
        __syncthreads();
        auto edge = [&](const Walk& w, int x) {
            const int p0 = w.prefix + (x - w.prefix) / w.nu * w.nu;
            return sp.snapped(x, p0, p0 + w.nu);
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
    const bool split = NB > 1 && a.bt_log2 == 4;   // a unit lies in two blocks
    uint8_t* ring = smem + warp * NS * kFewSlot<DP>;
    float* merge = reinterpret_cast<float*>(smem + W * NS * kFewSlot<DP>);
    // ---- copies: unit iu of piece iw is the next to be copied; the numbers of
    // its blocks are read one unit ahead
    Walk iw = cw;
    iw.hi = 0;
    bool more = true;
    int iu = 0, blk[NB];
    auto lookup = [&]() {
        while (more && iu >= iw.hi) {
            more = next_piece(iw);
            iu = iw.lo + warp;
        }
        if (!more) return;
        const int32_t* row = a.table + (size_t)iw.b * a.table_stride + (iu * UK >> a.bt_log2);
        // (a unit of two blocks may end in its first, and its first may lie before the window:
        // such a block may be gone, and the other's codes come in its place)
#pragma unroll
        for (int i = 0; i < NB; ++i)
            blk[i] = row[!split || iu * UK + i * 16 >= iw.s.start + iw.s.n ? 0
                         : iu * UK + i * 16 + 16 <= first_key(a, iw.s.start) ? 1 : i];
    };
    auto copy = [&](int to) {   // always closes a group, maybe an empty one
        if (more) {
            const uint32_t dst = smem_u32(ring) + to * kFewSlot<DP>;
#pragma unroll
            for (int i = 0; i < NB; ++i) {   // a block's part of the unit; with large blocks all of it
                if (i && !split) break;
                if ((uint32_t)blk[i] >= a.n_blocks) {
                    if (lane == 0) atomicOr(err, (unsigned)GRAFT_KV_EBLOCK);
                    blk[i] = 0;
                }
                const size_t bh = (size_t)blk[i] * H + iw.h;
                const size_t off = bh * (D << a.bt_log2) +
                                   ((iu * UK) & ((1 << a.bt_log2) - 1)) * D + lane * 16;
                const uint8_t *pk = a.k + off, *pv = a.v + off;
                const uint32_t part = dst + i * 16 * D + lane * 16;
                const int bytes = (split ? 16 : UK) * D;
#pragma unroll
                for (int c = 0; c < UK * DP; c += 512) {
                    if (FULL ? (split && c >= 16 * DP) : c + lane * 16 >= bytes) break;
                    cp_async16(part + c, pk + c);
                    cp_async16(part + UK * DP + c, pv + c);
                }
                if (lane < 2)
                    cp_async4(dst + 2 * UK * DP + i * 8 + lane * 4, (lane ? a.v_scale : a.k_scale) + bh);
            }
            iu += W;
            lookup();
        }
        cp_async_commit();
    };
    int slot = 0;   // of the warp's next unit
    FewState<DP, NT> st;
    uint32_t qf[CH][NT][8];
    float cn[NT][2];    // scale log2(e) of the columns' rows
    int pn[NT][2];      // positions of the columns' tokens

    // ---- two elements of a row of a finished pair, L relative to 2^M
    const int je = warp & 3, ce = (warp >> 2) & 1;   // the thread's accumulators: tile 4i + je, column ce
    auto finish = [&](int n, int i, float x0, float x1, float M, float L) {
        const int r = 8 * n + 2 * t + ce, d = 64 * i + 8 * g + 2 * je;
        const int tok = cw.s.n == 1 ? 0 : r / (int)a.group, head = r - tok * (int)a.group;
        if (tok >= cw.s.n || head >= (int)a.group || (!FULL && d >= D)) return;
        const int hq = cw.h * (int)a.group + head;
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
        x0 *= fo, x1 *= fo;
        uint16_t* y = (uint16_t*)a.out + (size_t)(cw.s.c0 + tok) * a.o_tok + hq * a.o_head + d;
        *reinterpret_cast<uint32_t*>(y) = a.bf16 ? pack2<GRAFT_BF16>(x0, x1) : pack2<GRAFT_F16>(x0, x1);
        if (a.lse && i == 0 && je == 0 && g == 0)
            a.lse[(size_t)(cw.s.c0 + tok) * a.q_heads + hq] = L != 0.f ? (ref + lg2(L)) * kLn2 : -INFINITY;
    };

    // ---- a pair's queries as B operands
    auto load_queries = [&]() {
        const int R = cw.s.n * (int)a.group;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = 8 * n + g;
            const bool on = r < R;
            const int tok = on && cw.s.n > 1 ? r / (int)a.group : 0;
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
                pn[n][c2] = cw.s.start + (cw.s.n > 1 ? min(8 * n + 2 * t + c2, R - 1) / (int)a.group : 0);
        }
    };

    lookup();
#pragma unroll 1
    for (int i = 0; i < NS; ++i) copy(i);
    while (next_piece(cw)) {
        st.reset();
        const int len = cw.s.start + cw.s.n;
        const int free_lo = first_key(a, len - 1);   // keys [free_lo, start] are seen by every row
        const int first = first_key(a, cw.s.start);  // keys before it by none
#pragma unroll 1
        for (int u = cw.lo + warp; u < cw.hi; u += W) {
            if (u < cw.lo + W) load_queries();
            const int key0 = u * UK;
            uint8_t* sl = ring + slot * kFewSlot<DP>;
            cp_async_wait<NS - 1>();
            __syncwarp();
            const bool edge_unit = key0 < free_lo || key0 + UK - 1 > cw.s.start;
            const int valid = len - key0;   // (at least 1)
            const float* sc = reinterpret_cast<const float*>(sl + 2 * UK * DP);
            if (FMT == GRAFT_KV_E4M3 && valid < UK) {
                // what lies after the last token may be NaN codes: 0 * NaN is no weight
                uint8_t* vr = sl + UK * DP;
                for (int i = valid * D / 16 + lane; i < UK * D / 16; i += 32)
                    reinterpret_cast<uint4*>(vr)[i] = make_uint4(0, 0, 0, 0);
                __syncwarp();
            }
            if (NB > 1 && FMT == GRAFT_KV_E4M3 && split && key0 + 16 <= first) {
                // .. and so may the codes that stand for a block before the window
                for (int i = lane; i < D; i += 32)
                    reinterpret_cast<uint4*>(sl + UK * DP)[i] = make_uint4(0, 0, 0, 0);
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
                const int blk = split ? kt : 0;
                const bool in = kt * 16 < valid;   // else no such block was copied
                const float ks = in ? sc[2 * blk] : 0.f;
                const float vs = in ? fmaxf(sc[2 * blk + 1], kKVScaleFloor) : 1.f;
                const float lv = lg2(vs);
                ivs[kt] = ex2(-lv);   // (what the weights are multiplied by, undone)
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
            // ---- reference for the exponents, weights, their sum.  The reference
            // (kPShift below the maximum it was taken from) follows only when a score
            // passes that maximum by more than kPSlack, which after the first units is
            // rare: no reduction across the lanes is needed for a unit that stays below.
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float mx[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    mx[c] = fmaxf(s[0][n][c], s[0][n][c + 2]);
#pragma unroll
                    for (int kt = 1; kt < KT; ++kt)
                        mx[c] = fmaxf(mx[c], fmaxf(s[kt][n][c], s[kt][n][c + 2]));
                }
                constexpr float limit = kPShift + kPSlack;
                if (__any_sync(~0u, mx[0] - st.m[n][0] > limit || mx[1] - st.m[n][1] > limit)) {
                    float f[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1)
                            mx[c] = fmaxf(mx[c], __shfl_xor_sync(~0u, mx[c], o));
                        const float up = fmaxf(st.m[n][c], reference(mx[c], kPShift));
                        f[c] = ex2(st.m[n][c] - up);
                        st.l[n][c] *= f[c];
                        st.m[n][c] = up;
                    }
#pragma unroll
                    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) st.o[i][n][e] *= f[e & 1];
                }
                const float b0 = st.m[n][0], b1 = st.m[n][1];
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
            copy(slot);
            slot = slot + 1 == NS ? 0 : slot + 1;
        }
        // ---- the lanes of a column hold sums over their own keys
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int o = 4; o < 32; o <<= 1)
                    st.l[n][c] += __shfl_xor_sync(~0u, st.l[n][c], o);
        // ---- the warps meet: every thread adds up two elements of each row tile
        const int active = min(W, cw.hi - cw.lo);
        constexpr int NO = kFewOut<DP, NT>;
        if (warp < active) {
            float* buf = merge + warp * NO * 32 + lane;
#pragma unroll
            for (int e = 0; e < NO; ++e) buf[e * 32] = (&st.o[0][0][0])[e];
            if (g == 0)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        sh_ml[warp][8 * n + 2 * t + c] = make_float2(st.m[n][c], st.l[n][c]);
        }
        __syncthreads();
        float M[NT], L[NT], x[NT][CH][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = 8 * n + 2 * t + ce;
            float f[W];
            M[n] = kNoMax, L[n] = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                f[w] = w < active ? sh_ml[w][r].x : kNoMax;
                M[n] = fmaxf(M[n], f[w]);
            }
#pragma unroll
            for (int i = 0; i < CH; ++i) x[n][i][0] = x[n][i][1] = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w)
                if (w < active) {
                    const float fw = ex2(f[w] - M[n]);
                    L[n] = fmaf(sh_ml[w][r].y, fw, L[n]);
#pragma unroll
                    for (int i = 0; i < CH; ++i) {
                        const float* e0 = merge + w * NO * 32 + (((4 * i + je) * NT + n) * 4 + ce) * 32 + lane;
                        x[n][i][0] = fmaf(e0[0], fw, x[n][i][0]);
                        x[n][i][1] = fmaf(e0[64], fw, x[n][i][1]);
                    }
                }
        }
        int ca, cb;
        sp.cuts(cw.p0, cw.p0 + cw.nu, ca, cb);
        if (cb >= ca) {   // pieces of the pair meet in the workspace
            const int first = ca - 1, pieces = cb - ca + 2;
            float* part = a.partials +
                          ((size_t)blockIdx.x * 2 + (cw.lo == cw.u0)) * kFewPartial<DP, NT>;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int i = 0; i < CH; ++i)
                    __stcg(reinterpret_cast<float2*>(part) + (n * CH + i) * kFewThreads + tid,
                           make_float2(x[n][i][0], x[n][i][1]));
                if (je == 0 && g == 0)
                    __stcg(reinterpret_cast<float2*>(part + NO * 32) + 8 * n + 2 * t + ce,
                           make_float2(M[n], L[n]));
            }
            __syncthreads();
            if (tid == 0) {
                // (release: the CTA's partial result before its count; acquire: the others')
                unsigned was;
                asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;"
                             : "=r"(was) : "l"(a.counters + first) : "memory");
                sh_last = was + 1 == (unsigned)pieces;
                if (sh_last) a.counters[first] = 0;
            }
            __syncthreads();
            if (!sh_last) continue;
            // the pair's last CTA adds up its pieces; piece k: CTA first + k
            const float* base = a.partials + (size_t)first * 2 * kFewPartial<DP, NT>;
            constexpr int KB = NT * CH == 1 ? 20 : NT * CH == 2 ? 10 : 4;   // pieces read at a time
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                M[n] = kNoMax, L[n] = 0.f;
#pragma unroll
                for (int i = 0; i < CH; ++i) x[n][i][0] = x[n][i][1] = 0.f;
            }
#pragma unroll 1
            for (int k0 = 0; k0 < pieces; k0 += KB) {
                float2 ml[KB][NT], v[KB][NT][CH];
#pragma unroll
                for (int k = 0; k < KB; ++k) {
                    const int kk = min(k0 + k, pieces - 1);
                    const float* p = base + (2 * kk + (kk == 0)) * kFewPartial<DP, NT>;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        ml[k][n] = __ldcg(reinterpret_cast<const float2*>(p + NO * 32) + 8 * n + 2 * t + ce);
#pragma unroll
                        for (int i = 0; i < CH; ++i)
                            v[k][n][i] = __ldcg(reinterpret_cast<const float2*>(p) + (n * CH + i) * kFewThreads + tid);
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float was = M[n];
#pragma unroll
                    for (int k = 0; k < KB; ++k) M[n] = fmaxf(M[n], ml[k][n].x);
                    const float f0 = ex2(was - M[n]);
                    L[n] *= f0;
#pragma unroll
                    for (int i = 0; i < CH; ++i) x[n][i][0] *= f0, x[n][i][1] *= f0;
#pragma unroll
                    for (int k = 0; k < KB; ++k) {
                        const float fk = k0 + k < pieces ? ex2(ml[k][n].x - M[n]) : 0.f;
                        L[n] = fmaf(ml[k][n].y, fk, L[n]);
#pragma unroll
                        for (int i = 0; i < CH; ++i) {
                            x[n][i][0] = fmaf(v[k][n][i].x, fk, x[n][i][0]);
                            x[n][i][1] = fmaf(v[k][n][i].y, fk, x[n][i][1]);
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < CH; ++i) finish(n, i, x[n][i][0], x[n][i][1], M[n], L[n]);
        __syncthreads();   // (before the next pair's states)
    }
    cp_async_wait<0>();
}

}  // namespace dev
}  // namespace graft
