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

}  // namespace dev
}  // namespace graft
