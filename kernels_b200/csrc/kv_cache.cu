// kv_cache.cu -- the paged 8-bit key/value cache: quantising tokens as they
// are written, and reading them back.
//
//   scale(block, head) = max(amax / qmax, 2^-64 [, old scale]),  code = round(x / scale)
//   value = code * scale
//
// Both kernels move each byte once and compute a few operations per element,
// so HBM bounds the long calls and launch plus load latency the short ones.
// Work items are the blocks that a sequence touches.  Writing gives each (item,
// head, K or V) a CTA: a block's amax, and the rounding again of its earlier codes
// when the scale grows, concern that CTA alone, so its elements stay in registers
// between the maximum and the rounding, and nothing is atomic.  Reading gives a
// CTA as many heads of an item as make 32 KB of codes.
// The item of a CTA follows from cu_tokens in closed form: sequence b's items
// start at cu_tokens[b] / block_tokens + 2 b, which leaves room for every
// block it can touch whatever its start, so no prefix sum of block counts is
// needed (a CTA past its sequence's blocks returns).
//
// Measured: reading 65521 tokens of 8 heads of 128 back in fp16 71 us, 5.7 TB/s; writing
// them 84 us, 4.8 TB/s (instruction issue, 67% of the slots: 13 warp instructions for 32 codes);
// the same in fp32 157 and 168 us, 4.3 and 4.0 TB/s; writing 7687 tokens of 8 heads of 64 and
// reading them back 14.0 us; one token of 64 sequences (8 heads of 128), written and its block
// read back, 7.6 us.
#include "rope.cuh"

#include <algorithm>

using namespace graft;
using namespace graft::dev;

namespace {

__device__ unsigned g_kv_err;

constexpr int kChunk = 8;        // elements a thread moves at once
constexpr int kWarpChunks = 256; // an item of up to so many chunks a head is a warp's (8 a lane)

struct KVArgs {
    uint8_t *k, *v;
    float *k_scale, *v_scale;
    const int32_t *table, *start, *cu;
    const void *x_k, *x_v;                 // rows (read by write, written by read)
    uint64_t tok_k, head_k, tok_v, head_v; // strides in elements
    uint32_t n_blocks, heads, bt, dim, n_seqs, table_stride, max_tokens, max_len, tokens;
    uint32_t bt_log2;
    uint32_t cpt, cpt_magic;   // chunks of a row; c / cpt = c cpt_magic >> 20 (c < 128 cpt <= 4096)
    uint32_t cta_heads;        // heads of a CTA (read)
    uint32_t wide;             // rows are 32-byte aligned (16-bit types; read)
};
// .. and of a write that turns the keys
struct KVRopeArgs : KVArgs {
    RopeArgs rope;
    const int32_t *positions, *rows, *count;   // or null
    const void* x_q;
    void* y_q;
    uint64_t tok_xq, head_xq, tok_yq, head_yq;
    uint32_t q_heads, cta_q_heads;             // query heads, and those of a CTA
    uint32_t q_ny;                             // CTAs of an item for its queries, the first ones
    uint32_t q_copy;                           // y_q is another buffer
};

// One item: `count` tokens of one sequence in one block.
struct Item {
    const int32_t* block;   // where the block's number stands
    int slot;               // first slot in it
    int row;                // row of the first token
    int count;
    int pos;                // position of the first token
};

// The item of flat index x (false: none).  Every thread of the CTA calls it.  The
// lengths of a sequence are read by the thread that looks at it, so that only one
// round trip to memory comes before the rows' and the block number's.
// counts: how many of each sequence's tokens are meant (null: all).
__device__ __forceinline__ bool find_item(const KVArgs& a, uint32_t x, Item& it,
                                          const int32_t* counts = nullptr) {
    __shared__ int sh_seq[5];   // sequence, its first row, one past its last, its start, its count
    const uint32_t bt = 1u << a.bt_log2;
    for (uint32_t s0 = 0;; s0 += blockDim.x) {
        const uint32_t s = s0 + threadIdx.x;
        bool here = false;   // x is one of its items: they start at or before x, the next one's after
        if (s < a.n_seqs) {
            const int c = a.cu[s], e = a.cu[s + 1], st = a.start[s];
            const int some = counts ? counts[s] : e - c;
            // (a sequence of fewer than no tokens may have no items that would tell; the last
            // CTA looks at every sequence up to the last or to one that it finds too long)
            if (e < c) atomicOr(&g_kv_err, (unsigned)GRAFT_KV_EBOUNDS);
            here = (s == 0 || ((uint32_t)c >> a.bt_log2) + 2 * s <= x) &&
                   (s + 1 == a.n_seqs || ((uint32_t)e >> a.bt_log2) + 2 * (s + 1) > x);
            if (here) sh_seq[0] = s, sh_seq[1] = c, sh_seq[2] = e, sh_seq[3] = st, sh_seq[4] = some;
        }
        const int found = __syncthreads_count(here);
        if (found == 1) break;
        // (none, or with cu_tokens that do not rise several: nothing to do here)
        if (found > 1 || s0 + blockDim.x >= a.n_seqs) return false;
    }
    const int b = sh_seq[0], c0 = sh_seq[1], all = sh_seq[2] - c0, n = counts ? sh_seq[4] : all;
    const int64_t start = sh_seq[3];
    if (c0 < 0 || n < 0 || n > all || n > (int)a.max_tokens || (uint64_t)c0 + (uint64_t)n > a.tokens ||
        start < 0 || (uint64_t)(start + n) > a.max_len) {
        if (threadIdx.x == 0) atomicOr(&g_kv_err, (unsigned)GRAFT_KV_EBOUNDS);
        return false;
    }
    if (n == 0) return false;
    const uint32_t j = x - (((uint32_t)c0 >> a.bt_log2) + 2 * b);
    const int64_t page = (start >> a.bt_log2) + j, base = page << a.bt_log2;
    if (base >= start + n) return false;
    const int64_t lo = base > start ? base : start;
    it.slot = (int)(lo - base);
    it.row = c0 + (int)(lo - start);
    it.pos = (int)lo;
    it.count = min((int)bt - it.slot, (int)(start + n - lo));
    it.block = a.table + (size_t)b * a.table_stride + (size_t)page;
    return true;
}
__device__ __forceinline__ bool good_block(const KVArgs& a, int block) {
    if ((uint32_t)block < a.n_blocks) return true;
    if (threadIdx.x == 0) atomicOr(&g_kv_err, (unsigned)GRAFT_KV_EBLOCK);
    return false;
}

// |x| of a finite element, 0 of another
__device__ __forceinline__ float fin_abs(float x) {
    const float a = fabsf(x);
    return a < __int_as_float(0x7f800000) ? a : 0.f;
}

// x / s for two finite x: the product with 1/s (correctly rounded) and one correction by the
// exact remainder, which gives the correctly rounded quotient (Markstein, 1990) in three
// operations instead of the general division's ten.
__device__ __forceinline__ uint64_t quotient2(uint64_t x, uint64_t minus_s, uint64_t inv) {
    const uint64_t q = mul2(x, inv);
    return fma2(fma2(q, minus_s, x), inv, q);
}

// Four quotients of finite elements as codes.  None is beyond qmax by more than its
// rounding, so an int8 code needs no clamp: the sum with 1.5 2^23 rounds to nearest even
// and holds the integer in its low bits.
template <int FMT>
__device__ __forceinline__ uint32_t finite_codes(uint64_t ab, uint64_t cd) {
    float a, b, c, d;
    if constexpr (FMT == GRAFT_KV_INT8) {
        const uint64_t k = pair(12582912.f, 12582912.f);
        unpair(add2(ab, k), a, b);
        unpair(add2(cd, k), c, d);
        return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040),
                           __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
    } else {
        unpair(ab, a, b);
        unpair(cd, c, d);
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
        return (uint32_t)hi << 16 | lo;
    }
}

// Eight elements as codes of scale s (inv: its reciprocal); odd: an infinity or a NaN may be among them.
template <int FMT>
__device__ __forceinline__ uint2 codes_of(const float (&f)[8], float s, uint64_t minus_s, uint64_t inv, bool odd) {
    uint2 o = make_uint2(0u, 0u);
    if (odd) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            o.x |= kv_code<FMT>(__fdiv_rn(f[e], s)) << (8 * e);
            o.y |= kv_code<FMT>(__fdiv_rn(f[e + 4], s)) << (8 * e);
        }
    } else {
        uint64_t q[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = quotient2(pair(f[2 * e], f[2 * e + 1]), minus_s, inv);
        o.x = finite_codes<FMT>(q[0], q[1]);
        o.y = finite_codes<FMT>(q[2], q[3]);
    }
    return o;
}

// A block's earlier `bytes` codes, times ratio (the old scale by the grown one).
template <int FMT>
__device__ __forceinline__ void round_again(uint8_t* codes, int bytes, float ratio, int tid, int T) {
    uint4* p = reinterpret_cast<uint4*>(codes);
#pragma unroll 4
    for (int c = tid; c < bytes / 16; c += T) {
        uint4 w = p[c];
        uint32_t* v = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float f[4];
            kv_decode4<FMT>(v[q], f);
            uint32_t o = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) o |= kv_code<FMT>(f[e] * ratio) << (8 * e);
            v[q] = o;
        }
        p[c] = w;
    }
}

// CH: chunks a thread holds.  WARP: each warp takes a (head, K or V) of the item,
// else the CTA takes one.
template <int DT, int FMT, int CH, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 512) kv_write_kernel(const __grid_constant__ KVArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ float red[16];
    Item it;
    if (!find_item(a, blockIdx.x, it)) return;
    const int block = *it.block;   // (not needed before the scale)
    const int unit = WARP ? blockIdx.y * 8 + (threadIdx.x >> 5) : blockIdx.y;
    if (WARP && unit >= 2 * (int)a.heads) return;
    const int head = unit >> 1;
    const bool is_v = unit & 1;
    const void* x = is_v ? a.x_v : a.x_k;
    const uint64_t ts = is_v ? a.tok_v : a.tok_k, hs = is_v ? a.head_v : a.head_k;
    const int tid = WARP ? threadIdx.x & 31 : threadIdx.x, T = WARP ? 32 : blockDim.x;
    const int n = it.count * (int)a.cpt;   // chunks of the item

    Raw<DT> r[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = tid + i * T;
        if (c < n) {
            const int t = (c * a.cpt_magic) >> 20;
            r[i] = load_raw<DT>(x, (it.row + t) * ts + head * hs + (c - t * (int)a.cpt) * kChunk);
        }
    }
    if (!good_block(a, block)) return;
    const size_t bh = (size_t)block * a.heads + head;
    uint8_t* codes = (is_v ? a.v : a.k) + bh * a.bt * a.dim;
    float* scale = (is_v ? a.v_scale : a.k_scale) + bh;
    const float old = it.slot ? *scale : 0.f;
    // ---- the largest magnitude.  16-bit floats without their sign are ordered like
    // integers, two to a word, infinities and NaN above all others.
    float amax = 0.f;
    bool odd = false;   // an infinity or a NaN among the thread's elements
    if constexpr (DT == GRAFT_F32) {
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (tid + i * T < n) {
                float f[8];
                to_floats<DT>(r[i], f);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    odd |= !(fabsf(f[e]) < INFINITY);
                    amax = fmaxf(amax, fabsf(f[e]));
                }
            }
    } else {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (tid + i * T < n) {
                const uint32_t* w = reinterpret_cast<const uint32_t*>(r[i].w);
#pragma unroll
                for (int e = 0; e < 4; ++e) m = __vmaxu2(m, w[e] & 0x7FFF7FFFu);
            }
        const uint32_t top = max(m & 0xFFFFu, m >> 16);
        odd = top >= (DT == GRAFT_F16 ? 0x7C00u : 0x7F80u);
        amax = DT == GRAFT_F16 ? h2f((uint16_t)top) : bf2f((uint16_t)top);
    }
    if (odd) {
        amax = 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (tid + i * T < n) {
                float f[8];
                to_floats<DT>(r[i], f);
#pragma unroll
                for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fin_abs(f[e]));
            }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, o));
    if constexpr (!WARP) {
        if ((tid & 31) == 0) red[tid >> 5] = amax;
        __syncthreads();
        for (int w = 0; w < T / 32; ++w) amax = fmaxf(amax, red[w]);
    }
    const float s = fmaxf(fmaxf(__fdiv_rn(amax, kKVQmax<FMT>), kKVScaleFloor), old);
    if constexpr (WARP) __syncwarp();   // (all lanes have read the old scale)
    if (tid == 0) *scale = s;
    const uint64_t inv = pair(__frcp_rn(s), __frcp_rn(s)), minus_s = pair(-s, -s);

    // the earlier tokens' codes, to the grown scale
    if (it.slot && s > old) round_again<FMT>(codes, it.slot * (int)a.dim, __fdiv_rn(old, s), tid, T);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = tid + i * T;
        if (c < n) {
            float f[8];
            to_floats<DT>(r[i], f);
            *reinterpret_cast<uint2*>(codes + (size_t)it.slot * a.dim + (size_t)c * kChunk) =
                codes_of<FMT>(f, s, minus_s, inv, odd);
        }
    }
}

// An item's queries: heads h0 .. of the CTA.  A thread takes a unit (16 elements) of a token for
// several heads, with the same sines and cosines.
template <int DT>
__device__ __forceinline__ void turn_queries(const KVRopeArgs& a, const Item& it, int h0) {
    const int units = a.dim / 16, per = it.count * units, T = blockDim.x;
    const int heads = min(a.cta_q_heads, a.q_heads - h0);
    const int G = max(1, min(heads, T / per));   // threads of a unit
    for (int i = threadIdx.x; i < per * G; i += T) {
        const int g = i / per, c = i - g * per, t = c / units, k = c - t * units;
        const bool turned = k < a.rope.pairs;
        if (!turned && !a.q_copy) continue;
        const int row = it.row + t;
        float cs[8], sn[8];
        if (turned)
            unit_turns<DT != GRAFT_F32>(a.rope, k, a.positions ? a.positions[row] : it.pos + t, cs, sn);
        const int e0 = unit_chunk(a.rope, k, 0) * 8, e1 = unit_chunk(a.rope, k, 1) * 8;
        constexpr int UN = DT == GRAFT_F32 ? 2 : 4;
        for (int j0 = g; j0 < heads; j0 += UN * G) {
            Raw<DT> p[UN], q[UN];
#pragma unroll
            for (int u = 0; u < UN; ++u)
                if (j0 + u * G < heads) {
                    const uint64_t from = row * a.tok_xq + (h0 + j0 + u * G) * a.head_xq;
                    p[u] = load_own<DT>(a.x_q, from + e0), q[u] = load_own<DT>(a.x_q, from + e1);
                }
#pragma unroll
            for (int u = 0; u < UN; ++u)
                if (j0 + u * G < heads) {
                    const uint64_t to = row * a.tok_yq + (h0 + j0 + u * G) * a.head_yq;
                    if (turned) {
                        float x[8], y[8];
                        to_floats<DT>(p[u], x), to_floats<DT>(q[u], y);
                        turn_unit(a.rope.half, cs, sn, x, y);
                        p[u] = from_floats<DT>(x), q[u] = from_floats<DT>(y);
                    }
                    store_raw<DT>(a.y_q, to + e0, p[u]), store_raw<DT>(a.y_q, to + e1, q[u]);
                }
        }
    }
}

// The same as kv_write_kernel with keys turned in fp32 before their maximum is taken.  A thread's
// chunks come in twos, the halves of a unit (rope.cuh), so that it holds both elements of its pairs.
// The first CTAs of an item turn its queries: 7687 tokens (64 query heads on 8 of 64) turned, written and
// read back 42 us, 46 with those CTAs last.  One token of 64 sequences and its block read back 9.7 us
// (7.6 without turning).  Registers bound the first (24 warps an SM), latency the second.
// (CTAs with 4 chunks a thread have 128 threads at most: the launch's rule.)
template <int DT, int FMT, int CH, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : CH == 4 ? 128 : 512, WARP ? (CH == 2 ? 3 : 2) : CH == 4 ? 6 : 1)
    kv_write_rope_kernel(const __grid_constant__ KVRopeArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ float red[16];
    Item it;
    if (!find_item(a, blockIdx.x, it, a.count)) return;
    if (blockIdx.y < a.q_ny) {
        turn_queries<DT>(a, it, blockIdx.y * a.cta_q_heads);
        return;
    }
    const int block = *it.block;   // (not needed before the scale)
    const int y = blockIdx.y - a.q_ny, unit = WARP ? y * 8 + (threadIdx.x >> 5) : y;
    if (WARP && unit >= 2 * (int)a.heads) return;
    const int head = unit >> 1;
    const bool is_v = unit & 1;
    const void* x = is_v ? a.x_v : a.x_k;
    const uint64_t ts = is_v ? a.tok_v : a.tok_k, hs = is_v ? a.head_v : a.head_k;
    const int tid = WARP ? threadIdx.x & 31 : threadIdx.x, T = WARP ? 32 : blockDim.x;
    const int upr = (int)a.cpt / 2, n = it.count * upr;   // units of a row, of the item

    float f[CH][8];
    int chunk[CH];
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < CH; i += 2) {
        const int w = tid + i / 2 * T;
        chunk[i] = -1;
        if (w < n) {
            const int t = (w * a.cpt_magic) >> 20, k = w - t * upr;
            int row = it.row + t;
            if (a.rows) row = a.rows[row];
            const bool turned = !is_v && k < a.rope.pairs;
            const int c0 = turned ? unit_chunk(a.rope, k, 0) : 2 * k, c1 = turned ? unit_chunk(a.rope, k, 1) : 2 * k + 1;
            chunk[i] = t * (int)a.cpt + c0, chunk[i + 1] = t * (int)a.cpt + c1;
            if ((uint32_t)row < a.tokens) {
                const uint64_t from = row * ts + head * hs;
                to_floats<DT>(load_raw<DT>(x, from + c0 * kChunk), f[i]);
                to_floats<DT>(load_raw<DT>(x, from + c1 * kChunk), f[i + 1]);
                if (turned) {
                    float cs[8], sn[8];
                    unit_turns<DT != GRAFT_F32>(a.rope, k, a.positions ? a.positions[row] : it.pos + t, cs, sn);
                    turn_unit(a.rope.half, cs, sn, f[i], f[i + 1]);
                }
            } else {
                atomicOr(&g_kv_err, (unsigned)GRAFT_KV_EBOUNDS);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[i][e] = f[i + 1][e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) amax = max_nan(amax, max_nan(fabsf(f[i][e]), fabsf(f[i + 1][e])));
        }
    }
    if (!good_block(a, block)) return;
    const size_t bh = (size_t)block * a.heads + head;
    uint8_t* codes = (is_v ? a.v : a.k) + bh * a.bt * a.dim;
    float* scale = (is_v ? a.v_scale : a.k_scale) + bh;
    const float old = it.slot ? *scale : 0.f;
    const bool odd = !(amax < INFINITY);
    if (odd) {
        amax = 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (chunk[i & ~1] >= 0)
#pragma unroll
                for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fin_abs(f[i][e]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, o));
    if constexpr (!WARP) {
        if ((tid & 31) == 0) red[tid >> 5] = amax;
        __syncthreads();
        for (int w = 0; w < T / 32; ++w) amax = fmaxf(amax, red[w]);
    }
    const float s = fmaxf(fmaxf(__fdiv_rn(amax, kKVQmax<FMT>), kKVScaleFloor), old);
    if constexpr (WARP) __syncwarp();   // (all lanes have read the old scale)
    if (tid == 0) *scale = s;
    const uint64_t inv = pair(__frcp_rn(s), __frcp_rn(s)), minus_s = pair(-s, -s);
    if (it.slot && s > old) round_again<FMT>(codes, it.slot * (int)a.dim, __fdiv_rn(old, s), tid, T);
#pragma unroll
    for (int i = 0; i < CH; ++i)
        if (chunk[i & ~1] >= 0)
            *reinterpret_cast<uint2*>(codes + (size_t)it.slot * a.dim + (size_t)chunk[i] * kChunk) =
                codes_of<FMT>(f[i], s, minus_s, inv, odd);
}

constexpr int kReadThreads = 256, kReadUnroll = 4;   // (kReadThreads: also the launch's)

template <int DT, int FMT>
__global__ void __launch_bounds__(kReadThreads) kv_read_kernel(const __grid_constant__ KVArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    Item it;
    if (!find_item(a, blockIdx.x, it)) return;
    const int block = *it.block;
    const int h0 = (blockIdx.y >> 1) * a.cta_heads, h1 = min(h0 + a.cta_heads, a.heads);
    const bool is_v = blockIdx.y & 1;
    void* y = const_cast<void*>(is_v ? a.x_v : a.x_k);
    const uint64_t ts = is_v ? a.tok_v : a.tok_k, hs = is_v ? a.head_v : a.head_k;
    const uint8_t* codes = is_v ? a.v : a.k;
    const float* scales = is_v ? a.v_scale : a.k_scale;
    if (!good_block(a, block)) return;
    const int per = it.count * (int)a.cpt, n = (h1 - h0) * per;   // chunks of 16 codes: a head's, all
    for (int c0 = threadIdx.x; c0 < n; c0 += kReadThreads * kReadUnroll) {
        uint4 w[kReadUnroll];
        float s[kReadUnroll];
        uint64_t to[kReadUnroll];
#pragma unroll
        for (int u = 0; u < kReadUnroll; ++u) {
            const int c = c0 + u * kReadThreads;
            if (c >= n) break;
            const int h = c / per, r = c - h * per, t = (r * a.cpt_magic) >> 20;
            const size_t bh = (size_t)block * a.heads + h0 + h;
            w[u] = ld_stream(codes + (bh * a.bt + it.slot) * a.dim + (size_t)r * 16);
            s[u] = scales[bh];
            to[u] = (it.row + t) * ts + (h0 + h) * hs + (r - t * (int)a.cpt) * 16;
        }
#pragma unroll
        for (int u = 0; u < kReadUnroll; ++u) {
            if (c0 + u * kReadThreads >= n) break;
            const uint32_t ws[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
            if constexpr (DT == GRAFT_F32) {
                float4* o = reinterpret_cast<float4*>((float*)y + to[u]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float f[4];
                    kv_decode4<FMT>(ws[i], f);
                    o[i] = make_float4(f[0] * s[u], f[1] * s[u], f[2] * s[u], f[3] * s[u]);
                }
            } else {
                uint32_t o[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float f[4];
                    kv_decode4<FMT>(ws[i], f);
                    o[2 * i] = pack2<DT>(f[0] * s[u], f[1] * s[u]);
                    o[2 * i + 1] = pack2<DT>(f[2] * s[u], f[3] * s[u]);
                }
                uint4* p = reinterpret_cast<uint4*>((uint16_t*)y + to[u]);
                if (a.wide) {   // whole 32-byte sectors
                    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p),
                                 "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]), "r"(o[5]),
                                 "r"(o[6]), "r"(o[7])
                                 : "memory");
                } else {
                    p[0] = make_uint4(o[0], o[1], o[2], o[3]);
                    p[1] = make_uint4(o[4], o[5], o[6], o[7]);
                }
            }
        }
    }
}

using KVKernel = void (*)(const KVArgs);
using KVRopeKernel = void (*)(const KVRopeArgs);
enum Form { kRead, kWriteOne, kWriteWarp, kWriteCta };   // kWriteOne: a chunk a lane
template <int DT, int FMT>
KVKernel pick(Form form, int chunks) {
    return form == kRead       ? kv_read_kernel<DT, FMT>
           : form == kWriteOne ? kv_write_kernel<DT, FMT, 1, true>
           : form == kWriteWarp ? kv_write_kernel<DT, FMT, 8, true>
           : chunks <= 4       ? kv_write_kernel<DT, FMT, 4, false>
                               : kv_write_kernel<DT, FMT, 8, false>;
}
template <int DT>
KVKernel pick(Form form, int chunks, uint32_t fmt) {
    return fmt == GRAFT_KV_INT8 ? pick<DT, GRAFT_KV_INT8>(form, chunks)
                                : pick<DT, GRAFT_KV_E4M3>(form, chunks);
}
template <int DT, int FMT>
KVRopeKernel pick_rope(Form form, int chunks) {
    return form == kWriteOne    ? kv_write_rope_kernel<DT, FMT, 2, true>
           : form == kWriteWarp ? kv_write_rope_kernel<DT, FMT, 8, true>
           : chunks <= 4        ? kv_write_rope_kernel<DT, FMT, 4, false>
                                : kv_write_rope_kernel<DT, FMT, 8, false>;
}
template <int DT>
KVRopeKernel pick_rope(Form form, int chunks, uint32_t fmt) {
    return fmt == GRAFT_KV_INT8 ? pick_rope<DT, GRAFT_KV_INT8>(form, chunks)
                                : pick_rope<DT, GRAFT_KV_E4M3>(form, chunks);
}

// turned: a write that turns the keys (its fields beyond KVArgs), or null
int kv_move(bool write, const GraftKVCache* cache, const GraftHeads* K, const GraftHeads* V,
            const GraftKVRange* range, KVRopeArgs* turned, cudaStream_t st) {
    int rc;
    if ((rc = kv_check_cache(cache)) || (rc = kv_check_range(cache, range)) ||
        (rc = kv_check_heads("K", K, cache->head_dim)) ||
        (rc = kv_check_heads("V", V, cache->head_dim)))
        return rc;
    GRAFT_REQUIRE(K->dtype == V->dtype && K->tokens == V->tokens,
                  "K and V must have the same type and number of tokens");
    if (range->n_seqs == 0 || K->tokens == 0) return GRAFT_OK;
    KVArgs a = {};
    a.k = (uint8_t*)cache->k, a.v = (uint8_t*)cache->v;
    a.k_scale = cache->k_scale, a.v_scale = cache->v_scale;
    a.table = range->block_table, a.start = range->start, a.cu = range->cu_tokens;
    a.x_k = K->data, a.x_v = V->data;
    a.tok_k = K->token_stride, a.head_k = K->head_stride;
    a.tok_v = V->token_stride, a.head_v = V->head_stride;
    a.n_blocks = cache->n_blocks, a.heads = cache->kv_heads, a.bt = cache->block_tokens;
    a.dim = cache->head_dim, a.n_seqs = range->n_seqs, a.table_stride = range->table_stride;
    a.max_tokens = range->max_tokens, a.max_len = range->max_len, a.tokens = K->tokens;
    const uint64_t bits = ((uint64_t)(uintptr_t)K->data | (uintptr_t)V->data |
                           2 * (K->token_stride | K->head_stride | V->token_stride | V->head_stride));
    a.wide = bits % 32 == 0;
    const uint64_t items = (uint64_t)K->tokens / a.bt + 2ull * a.n_seqs;
    GRAFT_REQUIRE(items < (1ull << 31), "too many tokens in one call");
    a.bt_log2 = a.bt == 16 ? 4 : a.bt == 32 ? 5 : a.bt == 64 ? 6 : 7;
    a.cpt = a.dim / (write ? kChunk : 16);
    a.cpt_magic = ((1u << 20) + a.cpt - 1) / a.cpt;
    a.cta_heads = std::min(a.heads, std::max(1u, 32768u / (a.bt * a.dim)));
    // Writing, a CTA a (head, K or V): 8 chunks of 8 elements a thread (what every thread does
    // once costs as much as two chunks), or 4 where that makes fewer than 128 threads.
    // 65521 tokens, blocks of 64, written and read back: 8 heads of 128 154 us so and 166 with
    // 4 chunks; 8 heads of 64 76 with 4 chunks (128 threads) and 78 with 8.  Where most CTAs
    // would be nearly empty and many, a warp each, eight to a CTA:
    //   one token of 64 sequences (8 heads of 128)      a chunk a lane 7.8 us, a CTA 10
    //   8 tokens of 256 sequences (8 heads of 64)       a warp 16.3 us, a CTA 22.0
    //   8 tokens of 64                                  a warp 10.3 us, a CTA 10.4
    //   32 tokens of one                                a warp 7.0 us, a CTA 5.8
    //   7687 tokens of 4, whole blocks of 16 (of 128)   a warp 22.6 us, a CTA 21.1
    const uint32_t most = std::min(range->max_tokens, a.bt) * a.cpt;   // chunks of an item
    DeviceInfo di;
    if (const int rc = current_device_info(&di)) return rc;
    const bool sparse = 2 * (uint64_t)range->max_tokens <= a.bt &&
                        items * 2 * a.heads > 16ull * di.sm_count;
    const Form form = !write                                ? kRead
                      : most <= 32                          ? kWriteOne
                      : most <= kWarpChunks && sparse       ? kWriteWarp
                                                            : kWriteCta;
    const int whole = (int)(a.bt * a.cpt);
    const int fourth = (whole / 4 + 31) / 32 * 32, eighth = (whole / 8 + 31) / 32 * 32;
    const int threads = form != kWriteCta
                            ? 256 : std::min(512, std::max({64, eighth, std::min(fourth, 128)}));
    const int chunks = (int)(a.bt * a.cpt + threads - 1) / threads;
    const uint32_t ny = form == kRead      ? 2 * ((a.heads + a.cta_heads - 1) / a.cta_heads)
                        : form == kWriteCta ? 2 * a.heads : (2 * a.heads + 7) / 8;
    if (turned) {
        *static_cast<KVArgs*>(turned) = a;
        KVRopeArgs& r = *turned;
        const uint32_t upr = r.cpt / 2;
        r.cpt_magic = ((1u << 20) + upr - 1) / upr;
        // queries: about 16 units a thread; these CTAs first, for they take the longest
        uint32_t q_ny = 0;
        if (r.x_q) {
            const uint64_t units = (uint64_t)std::min(range->max_tokens, a.bt) * (a.dim / 16) * r.q_heads;
            q_ny = (uint32_t)std::min<uint64_t>(r.q_heads, std::max<uint64_t>(1, units / (16ull * threads)));
            r.cta_q_heads = (r.q_heads + q_ny - 1) / q_ny;
            q_ny = (r.q_heads + r.cta_q_heads - 1) / r.cta_q_heads;
        }
        r.q_ny = q_ny;
        GRAFT_REQUIRE(ny + q_ny <= 65535, "too many heads in one call");
        const KVRopeKernel kern = K->dtype == GRAFT_F16    ? pick_rope<GRAFT_F16>(form, chunks, cache->format)
                                  : K->dtype == GRAFT_BF16 ? pick_rope<GRAFT_BF16>(form, chunks, cache->format)
                                                           : pick_rope<GRAFT_F32>(form, chunks, cache->format);
        return launch_pdl("kv_write_rope", kern, dim3((unsigned)items, ny + q_ny), threads, 0, st, r);
    }
    const KVKernel kern = K->dtype == GRAFT_F16    ? pick<GRAFT_F16>(form, chunks, cache->format)
                          : K->dtype == GRAFT_BF16 ? pick<GRAFT_BF16>(form, chunks, cache->format)
                                                   : pick<GRAFT_F32>(form, chunks, cache->format);
    return launch_pdl(write ? "kv_write" : "kv_read", kern,
                      dim3((unsigned)items, ny), threads, 0, st, a);
}

}  // namespace

namespace graft {

int kv_check_cache(const GraftKVCache* c) {
    clear_error();
    GRAFT_REQUIRE(c, "cache is null");
    GRAFT_REQUIRE(c->k && c->v && c->k_scale && c->v_scale, "the cache has a null buffer");
    GRAFT_REQUIRE(aligned(c->k, 16) && aligned(c->v, 16), "cache codes must be 16-byte aligned");
    GRAFT_REQUIRE(aligned(c->k_scale, 4) && aligned(c->v_scale, 4),
                  "cache scales must be 4-byte aligned");
    GRAFT_REQUIRE(c->format == GRAFT_KV_INT8 || c->format == GRAFT_KV_E4M3,
                  "unknown cache format %u", c->format);
    const uint32_t bt = c->block_tokens;
    GRAFT_REQUIRE(bt == 16 || bt == 32 || bt == 64 || bt == 128,
                  "block_tokens must be 16, 32, 64 or 128, not %u", bt);
    GRAFT_REQUIRE(c->head_dim >= 16 && c->head_dim <= 256 && c->head_dim % 16 == 0,
                  "head_dim must be a multiple of 16 up to 256, not %u", c->head_dim);
    GRAFT_REQUIRE(c->kv_heads >= 1 && c->kv_heads <= 32767, "kv_heads %u out of range",
                  c->kv_heads);
    GRAFT_REQUIRE(c->n_blocks >= 1 && c->n_blocks <= 0x7FFFFFFFu, "n_blocks %u out of range",
                  c->n_blocks);
    return GRAFT_OK;
}

int kv_check_range(const GraftKVCache* c, const GraftKVRange* r) {
    GRAFT_REQUIRE(r, "range is null");
    if (r->n_seqs == 0) return GRAFT_OK;
    GRAFT_REQUIRE(r->block_table && r->start && r->cu_tokens, "the range has a null array");
    GRAFT_REQUIRE(aligned(r->block_table, 4) && aligned(r->start, 4) && aligned(r->cu_tokens, 4),
                  "the range's arrays must be 4-byte aligned");
    GRAFT_REQUIRE(r->n_seqs < (1u << 28), "n_seqs %u out of range", r->n_seqs);
    GRAFT_REQUIRE(r->max_len <= 0x7FFFFFFFu && r->max_tokens <= r->max_len,
                  "max_tokens %u must not exceed max_len %u", r->max_tokens, r->max_len);
    GRAFT_REQUIRE((uint64_t)r->table_stride * c->block_tokens >= r->max_len,
                  "a block table row of %u blocks of %u tokens does not hold max_len %u",
                  r->table_stride, c->block_tokens, r->max_len);
    return GRAFT_OK;
}

int kv_check_heads(const char* name, const GraftHeads* h, uint32_t dim) {
    GRAFT_REQUIRE(h, "%s is null", name);
    GRAFT_REQUIRE(h->dtype == GRAFT_F16 || h->dtype == GRAFT_BF16 || h->dtype == GRAFT_F32,
                  "%s: unknown element type %u", name, h->dtype);
    if (h->tokens == 0) return GRAFT_OK;
    const uint64_t es = h->dtype == GRAFT_F32 ? 4 : 2;
    GRAFT_REQUIRE(h->data && aligned(h->data, 16), "%s must be a 16-byte aligned buffer", name);
    GRAFT_REQUIRE(h->token_stride * es % 16 == 0 && h->head_stride * es % 16 == 0,
                  "%s: strides must be multiples of 16 bytes", name);
    GRAFT_REQUIRE(h->tokens <= 0x7FFFFFFFu, "%s: too many tokens", name);
    (void)dim;
    return GRAFT_OK;
}

unsigned kv_cache_device_errors(bool clear) { return read_device_errors(g_kv_err, clear); }

}  // namespace graft

extern "C" int graft_kv_write(const GraftKVCache* cache, const GraftHeads* K, const GraftHeads* V,
                              const GraftKVRange* range, graft_stream_t stream) {
    return kv_move(true, cache, K, V, range, nullptr, stream);
}

extern "C" int graft_kv_write_rope(const GraftKVCache* cache, const GraftHeads* K, const GraftHeads* V,
                                   const GraftKVRange* range, const GraftRope* rope,
                                   const int32_t* positions, const int32_t* rows, const int32_t* count,
                                   const GraftHeads* q, const GraftHeads* q_out, uint32_t q_heads,
                                   graft_stream_t stream) {
    int rc;
    if ((rc = kv_check_cache(cache)) || (rc = check_rope(rope, cache->head_dim))) return rc;
    GRAFT_REQUIRE(aligned(positions, 4) && aligned(rows, 4) && aligned(count, 4),
                  "positions, rows and count must be 4-byte aligned");
    GRAFT_REQUIRE(!rows == !count, "rows and count go together");
    GRAFT_REQUIRE(!q == !q_out, "q and q_out go together");
    KVRopeArgs a = {};
    a.rope = rope_args(rope);
    a.positions = positions, a.rows = rows, a.count = count;
    if (q) {
        GRAFT_REQUIRE(!rows, "q cannot be turned together with rows and count");
        GRAFT_REQUIRE(K, "K is null");
        if ((rc = check_rope_rows(q, q_out, q_heads))) return rc;
        GRAFT_REQUIRE(q->dtype == K->dtype && q->tokens == K->tokens,
                      "q and K must have the same type and number of tokens");
        if (q_heads) {
            a.x_q = q->data, a.y_q = q_out->data;
            a.tok_xq = q->token_stride, a.head_xq = q->head_stride;
            a.tok_yq = q_out->token_stride, a.head_yq = q_out->head_stride;
            a.q_heads = q_heads, a.q_copy = q->data != q_out->data;
        }
    }
    return kv_move(true, cache, K, V, range, &a, stream);
}

extern "C" int graft_kv_read(const GraftKVCache* cache, const GraftHeads* K, const GraftHeads* V,
                             const GraftKVRange* range, graft_stream_t stream) {
    return kv_move(false, cache, K, V, range, nullptr, stream);
}

extern "C" int graft_kv_device_errors(uint32_t* bits, int clear) {
    clear_error();
    GRAFT_REQUIRE(bits, "bits pointer is null");
    GRAFT_CUDA(cudaDeviceSynchronize());
    *bits = kv_cache_device_errors(clear != 0) | attn_device_errors(clear != 0) |
            tree_device_errors(clear != 0);
    return GRAFT_OK;
}
