// attn_common.cuh -- what the attention kernels over the 8-bit cache share:
// arguments, code conversions to fp16 pairs, matrix instructions, the split of
// the work over the grid and the joining of partial results.
#pragma once
#include "attn_split.cuh"
#include "kv_common.cuh"

namespace graft {
namespace dev {

struct AttnArgs {
    const uint8_t *k, *v;
    const float *k_scale, *v_scale;
    const int32_t *table, *start, *cu;
    const void* q;
    void* out;
    const float* sinks;
    float* lse;
    uint64_t q_tok, q_head, o_tok, o_head;
    uint32_t n_blocks, heads, bt, dim, n_seqs, table_stride, max_tokens, max_len, tokens;
    uint32_t q_heads, group, window;
    float scale;
    int bt_log2;          // block_tokens = 1 << bt_log2
    int bf16;             // q and out: 1 bf16, 0 fp16
    unsigned* counters;   // one per CTA, zero between calls
    float* partials;      // two slots per CTA
    int min_units;        // smallest share of a CTA that is worth one
    int pad_units;        // units that a pair costs besides its own
    // of trees of drafted tokens (TREE): which new tokens a token sees, and where it stands
    const uint32_t* mask;     // [tokens][mask_stride]
    uint64_t mask_stride;     // words
    const int32_t* positions; // with a window
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// The reference of a row without a key yet: finite, so that a masked score
// (-inf) minus it is -inf and never NaN.
constexpr float kNoMax = -1e30f;
// Weights are held as 2^(t - m) for a reference m that lies kPShift below the largest
// t that it was taken from, and that no t passes by more than kPShift + kPSlack: at most
// 2^14 in fp16, which keeps its 11 bits down to 2^-28 of that.
constexpr float kPShift = 10.f, kPSlack = 4.f;
// The reference `shift` below a score t.  Above 2^25 steps of fp32 are as large as the
// shift: where the difference would be rounded to more than shift + kPSlack, which fp16
// might not hold as an exponent, it is t itself.
__device__ __forceinline__ float reference(float t, float shift) {
    const float r = t - shift;
    return t - r > shift + kPSlack ? t : r;
}

// Limit of every wait for a kernel's own copies or products.
constexpr uint64_t kAttnWaitNs = 2000000000ull;
// Most CTAs of an attention grid: one counter and two partial slots each.
constexpr int kAttnMaxGrid = 512;
constexpr int kChunkMaxGrid = 192;   // of the kernel for many rows (two counters a CTA)

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Whether phase `parity` of a barrier has completed (does not suspend).
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// A sequence of the range as the attention kernels see it (n = 0: skip it).
struct Seq {
    int c0, n, start;
};
__device__ __forceinline__ Seq load_seq(const AttnArgs& a, int b, unsigned* err) {
    Seq s;
    s.c0 = a.cu[b];
    s.n = a.cu[b + 1] - s.c0;
    s.start = a.start[b];
    if (s.c0 < 0 || s.n < 0 || s.n > (int)a.max_tokens ||
        (uint64_t)s.c0 + (uint64_t)s.n > a.tokens || s.start < 0 ||
        (uint64_t)((int64_t)s.start + s.n) > a.max_len) {
        atomicOr(err, (unsigned)GRAFT_KV_EBOUNDS);
        s.n = 0;
    }
    return s;
}
// First key that token i (position p) sees.
__device__ __forceinline__ int first_key(const AttnArgs& a, int p) {
    return a.window && p >= (int)a.window ? p - (int)a.window + 1 : 0;
}

// .. in a tree, where all that is before the sequence's start is seen, or what its window leaves
__device__ __forceinline__ int first_tree_key(const AttnArgs& a, const Seq& s, int tok) {
    return a.window ? first_key(a, max(s.start, a.positions[s.c0 + tok])) : 0;
}
// Bits lo .. hi - 1 of 32, for any lo and hi.
__device__ __forceinline__ uint32_t bit_range(int lo, int hi) {
    const uint32_t below = hi >= 32 ? ~0u : hi <= 0 ? 0u : (1u << hi) - 1u;
    return lo <= 0 ? below : lo >= 32 ? 0u : below & ~((1u << lo) - 1u);
}
// Which of the 32 keys from `key` on a token of a tree sees: those in [lo, start) and those of its
// sequence's n new tokens whose bits are set in its mask.
__device__ __forceinline__ uint32_t seen32(const uint32_t* mask, const Seq& s, int lo, int key) {
    uint32_t w = bit_range(lo - key, s.start - key);
    const int at = key - s.start;   // the keys' place among the new tokens
    if (at > -32 && at < s.n) {
        uint32_t m;
        if (at < 0) {
            m = mask[0] << -at;
        } else {
            const int i = at >> 5;
            m = mask[i] >> (at & 31);
            if ((at & 31) && (i + 1) * 32 < s.n) m |= mask[i + 1] << (32 - (at & 31));
        }
        w |= m & bit_range(-at, s.n - at);
    }
    return w;
}

// ---- codes to fp16 pairs
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t s) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(s));
    return r;
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// The four codes of a word as fp16 pairs, codes 0,1 and 2,3.  An int8 code with
// its sign bit flipped is code + 128; as the low byte of 0x64xx that is the fp16
// number 1024 + 128 + code, and one exact subtraction of 1152 leaves the code.
template <int FMT>
__device__ __forceinline__ void codes_h2(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (FMT == GRAFT_KV_INT8) {
        w ^= 0x80808080u;
        lo = hsub2(prmt(w, 0x64646464u, 0x4140), 0x64806480u);
        hi = hsub2(prmt(w, 0x64646464u, 0x4342), 0x64806480u);
    } else {
        asm("{\n\t.reg .b16 a, b;\n\t"
            "mov.b32 {a, b}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
            "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    }
}

// D += A (16 x 16, fp16, row) B (16 x 8, fp16, col), fp32 sums
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 8 x 8 transpose of 16-bit elements across the warp
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Sixteen consecutive query elements as eight fp16 pairs.  bf16 queries become
// fp16 through a power of two per row that brings the row's largest magnitude
// to [2^14, 2^15): every element keeps its 8 bits unless it is under 2^-28 of
// the row's largest.  `up` multiplies the scores to undo it.
__device__ __forceinline__ float bf16_row_exponent(float amax) {
    if (!(amax > 0.f) || amax > 3.4e38f) return 0.f;   // zeros; NaN, infinity: as they are
    const int e = (int)(__float_as_uint(amax) >> 23) - 127 - 14;
    return (float)max(e, -126);
}

}  // namespace dev
}  // namespace graft
