// attn_split.cuh -- arithmetic of the attention kernels' split of the work.  Plain
// C++ that the host can run too (the tests do, against sums taken one by one).
#pragma once

#ifdef __CUDACC__
#define GRAFT_HD __host__ __device__ __forceinline__
#else
#define GRAFT_HD inline
#endif

namespace graft {
namespace dev {

// Keys that the first `rt` row tiles of `tt` tokens of a sequence see between them, each
// counted with `pad` more: row tile i covers tokens i tt .. min(n, (i + 1) tt) - 1 and its
// keys are those from its first token's first one to its last token's own.  `tiles`:
// all row tiles of the sequence's n tokens, of which the first is at position `start`.
// window 0: every key is seen; any other window, up to the largest int, with
// start + n <= 2^30.
GRAFT_HD long long tile_keys(int start, int n, int tt, int tiles, int rt, int window, int pad) {
    const long long c = rt;
    long long k = c * ((long long)start + pad) + c * (c + 1) / 2 * tt;
    if (rt == tiles) k -= c * tt - n;   // (the last tile may have fewer tokens)
    if (window) {   // first keys: start - window + 1 + tt i where that is positive
        const int first = start - window + 1;
        // (tt - 1 - first reaches 2^31 + 253: unsigned)
        const unsigned none = first >= 0 ? 0u : ((unsigned)(tt - 1) - (unsigned)first) / (unsigned)tt;
        const int skip = none < (unsigned)rt ? (int)none : rt;
        const long long r = rt - skip;
        k -= r * (first + (long long)skip * tt) + (r - 1) * r / 2 * tt;
    }
    return k;
}

// ---- the split of the work
// Units (fixed numbers of keys) of all (sequence, tile, head) "pairs" lie in
// one row, each pair preceded by `pad` empty ones that stand for what a pair
// costs besides its units (queries, joining the warps, output).  CTA c of G
// takes those from x_c to x_{c+1}, where the x_c cut the row evenly (the first
// U % G shares are one longer), each moved to its pair's edge if it would
// leave a piece of less than `snap` units.  A pair that is cut has as its first
// piece the CTA before the first cut, and each CTA holds at most one first
// piece and one later piece, so two partial slots and one counter per CTA are
// enough.  The few-row kernel counts in its units (U + pad + snap < 2^31, the host's check),
// the kernel for many rows in keys, whose sums over row tiles have a closed form.
template <typename T>
struct Split {
    T U, share;              // share = U / G, longer = U % G
    int G, pad, snap, longer;
    GRAFT_HD void set(T units, int ctas, int pad_units, int snap_units) {
        U = units, G = ctas, pad = pad_units, snap = snap_units;
        share = U / G, longer = (int)(U - share * G);
    }
    GRAFT_HD T bound(int c) const { return c * share + (c < longer ? c : longer); }
    // the first CTA whose bound is x or more (x > 0; the quotients' numerators stay below U)
    GRAFT_HD int at_least(T x) const {
        const T head = longer * (share + 1);
        return (int)(x <= head ? (x - 1) / (share + 1) + 1 : longer + (x - head - 1) / share + 1);
    }
    GRAFT_HD T snapped(T x, T p0, T p1) const {
        const bool head = x < p0 + pad + snap, tail = x > p1 - snap;
        return !head && !tail ? x : !tail || (head && x - p0 <= p1 - x) ? p0 : p1;
    }
    // cuts inside [p0, p1): CTAs ca..cb start there (none if cb < ca)
    GRAFT_HD void cuts(T p0, T p1, int& ca, int& cb) const {
        const T lo = p0 + pad + snap, hi = p1 - snap;
        ca = 0, cb = -1;
        if (lo > hi) return;
        ca = at_least(lo);
        cb = at_least(hi + 1) - 1;
    }
};

}  // namespace dev
}  // namespace graft
