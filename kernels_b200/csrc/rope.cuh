// rope.cuh -- rotary positions on the device: angles, and pairs of chunks turned in fp32.
//
// A frequency is held as a fraction of a turn in 64 bits, F = f / 2 pi * 2^64, so the
// product with a position, modulo 2^64, is the angle within the turn: exact whatever the
// position, where fp32 is off by 2^-24 of the whole angle (0.008 radians at 131072).
#pragma once
#include "kv_common.cuh"

namespace graft {

int check_rope(const GraftRope* r, uint32_t head_dim);
// x and out of a turn: the same rows, or other ones (out's own apart)
int check_rope_rows(const GraftHeads* x, const GraftHeads* y, uint32_t heads);

namespace dev {

// Amplitude times cosine and sine of pos * turns.  FAST: the device's approximate ones (off by
// 2^-21) of the angle to 2^-24 of a turn, for results of 11 bits or fewer; the angle's upper 23
// bits become a number in [1, 2) without a conversion.
template <bool FAST>
__device__ __forceinline__ void rope_turn(int pos, uint64_t turns, float amp, float amp_s, float& c,
                                          float& s) {
    const uint32_t at = (uint32_t)((uint64_t)(int64_t)pos * turns >> 32);
    if constexpr (FAST) {
        // (half a turn off: both signs change, and the angle lies in [-pi, pi))
        const float x = fmaf(__uint_as_float(0x3F800000u + ((at + 256u) >> 9)), 6.283185307f, -9.424777961f);
        c = -amp * __cosf(x), s = -amp_s * __sinf(x);
    } else {
        float sn, cs;
        sincospif((float)(int32_t)at * 0x1p-31f, &sn, &cs);
        c = amp * cs, s = amp_s * sn;
    }
}

struct RopeArgs {
    const uint64_t* turns;
    float amp, amp_s;   // of the cosine and of the sine (negative: turned back)
    int pairs;          // chunks of 8 pairs of a head, dims / 16
    int half;           // pairs are i, i + dims / 2 (else neighbours)
};

// Heads are cut into units of 16 elements, two chunks of 8: units k < pairs hold 8 pairs
// (half layout: chunks k and k + pairs; else 2k and 2k + 1), the others are not turned.
__device__ __forceinline__ int unit_chunk(const RopeArgs& r, int k, int second) {
    return r.half && k < r.pairs ? k + second * r.pairs : 2 * k + second;
}

// The unit's cosines and sines.
template <bool FAST>
__device__ __forceinline__ void unit_turns(const RopeArgs& r, int k, int pos, float (&c)[8], float (&s)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const ulonglong2 f = __ldg(reinterpret_cast<const ulonglong2*>(r.turns + 8 * k + i));
        rope_turn<FAST>(pos, f.x, r.amp, r.amp_s, c[i], s[i]);
        rope_turn<FAST>(pos, f.y, r.amp, r.amp_s, c[i + 1], s[i + 1]);
    }
}
// Its two chunks turned.
__device__ __forceinline__ void turn_unit(bool half, const float (&c)[8], const float (&s)[8], float (&a)[8],
                                          float (&b)[8]) {
    if (half) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = a[i], y = b[i];
            a[i] = fmaf(x, c[i], -(y * s[i])), b[i] = fmaf(y, c[i], x * s[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            float x = a[i], y = a[i + 1];
            a[i] = fmaf(x, c[i / 2], -(y * s[i / 2])), a[i + 1] = fmaf(y, c[i / 2], x * s[i / 2]);
            x = b[i], y = b[i + 1];
            b[i] = fmaf(x, c[4 + i / 2], -(y * s[4 + i / 2])), b[i + 1] = fmaf(y, c[4 + i / 2], x * s[4 + i / 2]);
        }
    }
}

// Chunks of 8 elements of a buffer.
template <int DT>
struct Raw {
    uint4 w[DT == GRAFT_F32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ Raw<DT> load_raw(const void* base, uint64_t elem) {
    Raw<DT> r;
    const char* p = (const char*)base + elem * (DT == GRAFT_F32 ? 4 : 2);
    r.w[0] = ld_stream(p);
    if constexpr (DT == GRAFT_F32) r.w[1] = ld_stream(p + 16);
    return r;
}
// .. of one that the kernel may write
template <int DT>
__device__ __forceinline__ Raw<DT> load_own(const void* base, uint64_t elem) {
    Raw<DT> r;
    const uint4* p = reinterpret_cast<const uint4*>((const char*)base + elem * (DT == GRAFT_F32 ? 4 : 2));
    r.w[0] = p[0];
    if constexpr (DT == GRAFT_F32) r.w[1] = p[1];
    return r;
}
template <int DT>
__device__ __forceinline__ void to_floats(const Raw<DT>& r, float (&f)[8]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(r.w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == GRAFT_F32) {
            f[2 * i] = __uint_as_float(w[2 * i]);
            f[2 * i + 1] = __uint_as_float(w[2 * i + 1]);
        } else {
            const float2 p = unpack2<DT>(w[i]);
            f[2 * i] = p.x, f[2 * i + 1] = p.y;
        }
    }
}
template <int DT>
__device__ __forceinline__ Raw<DT> from_floats(const float (&f)[8]) {
    Raw<DT> r;
    uint32_t* w = reinterpret_cast<uint32_t*>(r.w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == GRAFT_F32) {
            w[2 * i] = __float_as_uint(f[2 * i]), w[2 * i + 1] = __float_as_uint(f[2 * i + 1]);
        } else {
            w[i] = pack2<DT>(f[2 * i], f[2 * i + 1]);
        }
    }
    return r;
}
template <int DT>
__device__ __forceinline__ void store_raw(void* base, uint64_t elem, const Raw<DT>& r) {
    uint4* p = reinterpret_cast<uint4*>((char*)base + elem * (DT == GRAFT_F32 ? 4 : 2));
    p[0] = r.w[0];
    if constexpr (DT == GRAFT_F32) p[1] = r.w[1];
}

}  // namespace dev

dev::RopeArgs rope_args(const GraftRope* r);

}  // namespace graft
