// kv_common.cuh -- what the 8-bit key/value cache's kernels share: the device
// view of a cache and a token range, code conversions, argument checks.
#pragma once
#include "async_copy.cuh"
#include "graft_common.cuh"

namespace graft {

// Checks of the public structs (GRAFT_EINVAL with a message).
int kv_check_cache(const GraftKVCache* c);
int kv_check_range(const GraftKVCache* c, const GraftKVRange* r);
int kv_check_heads(const char* name, const GraftHeads* h, uint32_t dim);

unsigned kv_cache_device_errors(bool clear);
unsigned attn_device_errors(bool clear);
unsigned tree_device_errors(bool clear);

// Reads (and resets) one kernel file's device error word.
template <typename Symbol>
unsigned read_device_errors(const Symbol& sym, bool clear) {
    unsigned v = 0;
    if (cudaMemcpyFromSymbol(&v, sym, sizeof v) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    if (clear && v) {
        const unsigned z = 0;
        cudaMemcpyToSymbol(sym, &z, sizeof z);
    }
    return v;
}

// Launches a kernel that calls griddepcontrol.wait before it touches memory.
template <typename... K, typename... A>
int launch_pdl(const char* what, void (*kern)(K...), dim3 grid, int threads, int smem,
               cudaStream_t st, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
    if (e != cudaSuccess) {
        cudaGetLastError();
        set_error("%s: launch failed: %s", what, cudaGetErrorString(e));
        return GRAFT_ECUDA;
    }
    return check_launch(what);
}

namespace dev {

// Smallest scale that is stored: blocks of zeros need no special case, and
// log2 of a scale stays far from fp32's limits.
constexpr float kKVScaleFloor = 5.421010862427522e-20f;   // 2^-64

template <int FMT>
constexpr float kKVQmax = FMT == GRAFT_KV_INT8 ? 127.f : 448.f;

// x / scale (already divided) to a code byte: nearest even, saturating, NaN to 0.
template <int FMT>
__device__ __forceinline__ uint32_t kv_code(float y) {
    if constexpr (FMT == GRAFT_KV_INT8) {
        const int q = __float2int_rn(y);   // NaN gives 0, infinities saturate
        return (uint32_t)max(-127, min(127, q)) & 0xFFu;
    } else {
        y = (y == y) ? y : 0.f;
        uint16_t r;   // low byte: the second operand
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(y));
        return r & 0xFFu;
    }
}

// Four codes of a word to fp32.
template <int FMT>
__device__ __forceinline__ void kv_decode4(uint32_t w, float (&f)[4]) {
    if constexpr (FMT == GRAFT_KV_INT8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = (float)(int8_t)(w >> (8 * i));
    } else {
        uint32_t lo, hi;
        asm("{\n\t.reg .b16 a, b;\n\t"
            "mov.b32 {a, b}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
            "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
        const float2 x = __half22float2(*reinterpret_cast<__half2*>(&lo));
        const float2 y = __half22float2(*reinterpret_cast<__half2*>(&hi));
        f[0] = x.x, f[1] = x.y, f[2] = y.x, f[3] = y.y;
    }
}

// Two 16-bit elements of a word to fp32 (DT: GRAFT_F16 or GRAFT_BF16).
template <int DT>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (DT == GRAFT_F16) return __half22float2(*reinterpret_cast<__half2*>(&w));
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (DT == GRAFT_F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float max_nan(float a, float b) {   // a NaN stays one
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// Pairs of fp32 numbers (sm_100's two-wide operations).
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t x, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

}  // namespace dev
}  // namespace graft
