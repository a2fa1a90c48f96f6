// logits.cuh -- rows of logits as the kernels over them read them: chunks of 16 bytes
// at any alignment, differences and maxima without conversions, keys that order.
#pragma once
#include "kv_common.cuh"

namespace graft {
namespace dev {

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// fp32 in the order of unsigned integers (finite and infinite; -0 = +0)
__device__ __forceinline__ uint32_t order(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float unorder(uint32_t o) {
    return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) {
    return ((uint64_t)order(x) << 32) | (0xFFFFFFFFu - index);
}

template <int DT>
__device__ __forceinline__ float logit(const void* row, uint32_t i) {
    if constexpr (DT == GRAFT_F32) return ((const float*)row)[i];
    const uint16_t w = ((const uint16_t*)row)[i];
    return DT == GRAFT_F16 ? h2f(w) : bf2f(w);
}
template <int DT>
constexpr int kPer = DT == GRAFT_F32 ? 4 : 8;   // elements of a chunk

// A chunk that begins `first` elements into a row and lies partly outside it; elements
// outside are -inf and are not read.
template <int DT>
__device__ __noinline__ uint4 edge_chunk(const void* row, int first, uint32_t vocab) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == GRAFT_F32) {
            const int e = first + i;
            w[i] = e >= 0 && e < (int)vocab ? ((const uint32_t*)row)[e] : 0xFF800000u;
        } else {
            const uint32_t none = DT == GRAFT_F16 ? 0xFC00u : 0xFF80u;
            const int e = first + 2 * i;
            w[i] = (e >= 0 && e < (int)vocab ? ((const uint16_t*)row)[e] : none) |
                   (e + 1 >= 0 && e + 1 < (int)vocab ? ((const uint16_t*)row)[e + 1] : none) << 16;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// Chunk c of a row whose first element is `off` elements into the row's first 16-byte chunk.
template <int DT>
__device__ __forceinline__ uint4 load_chunk(const void* row, int off, uint32_t vocab, int c) {
    constexpr int N = kPer<DT>;
    const int first = c * N - off;
    if (first >= 0 && first + N <= (int)vocab)
        return ld_stream((const char*)row + (int64_t)first * (16 / N));
    return edge_chunk<DT>(row, first, vocab);
}
template <int DT>
__device__ __forceinline__ void floats_of(const uint4& v, float (&x)[kPer<DT>]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == GRAFT_F32) {
            x[i] = __uint_as_float(w[i]);
        } else {
            const float2 p = unpack2<DT>(w[i]);
            x[2 * i] = p.x, x[2 * i + 1] = p.y;
        }
    }
}

// Two 16-bit logits minus ref in fp32: fma.rn.f32.f16 with a factor of one, so
// that no conversion is needed.
template <int DT>
__device__ __forceinline__ void minus(uint32_t w, float ref, float& d0, float& d1) {
    if constexpr (DT == GRAFT_F16) {
        asm("{\n\t.reg .f16 a, b, one;\n\t"
            "mov.b32 {a, b}, %2;\n\tmov.b16 one, 0x3C00;\n\t"
            "fma.rn.f32.f16 %0, a, one, %3;\n\tfma.rn.f32.f16 %1, b, one, %3;\n\t}"
            : "=f"(d0), "=f"(d1) : "r"(w), "f"(-ref));
    } else {
        asm("{\n\t.reg .b16 a, b, one;\n\t"
            "mov.b32 {a, b}, %2;\n\tmov.b16 one, 0x3F80;\n\t"
            "fma.rn.f32.bf16 %0, a, one, %3;\n\tfma.rn.f32.bf16 %1, b, one, %3;\n\t}"
            : "=f"(d0), "=f"(d1) : "r"(w), "f"(-ref));
    }
}

// Largest element of a chunk (NaN is passed over).
template <int DT>
__device__ __forceinline__ float chunk_max(const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if constexpr (DT == GRAFT_F32) {
        return fmaxf(fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1])),
                     fmaxf(__uint_as_float(w[2]), __uint_as_float(w[3])));
    } else {
        uint32_t m = w[0];
#pragma unroll
        for (int i = 1; i < 4; ++i) {
            if constexpr (DT == GRAFT_F16) asm("max.f16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i]));
            else asm("max.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i]));
        }
        const float2 p = unpack2<DT>(m);
        return fmaxf(p.x, p.y);
    }
}

}  // namespace dev
}  // namespace graft
