// logprobs.cu -- log probability of a given token, entropy and the top
// alternatives of each row of logits.
//
//   z = scale*logit, lse = log sum exp z, logprob = z[target] - lse,
//   entropy = lse - sum p z
//
// One CTA per row: a pass for the maximum, one for the sums, and one for each
// alternative (the largest logit after the one before it).
#include "kv_common.cuh"

#include <cmath>

using namespace graft;
using namespace graft::dev;

namespace {

constexpr int kThreads = 512;
constexpr float kLog2e = 1.4426950408889634f;

struct LpArgs {
    const void* logits;
    const int32_t* targets;
    float *logprob, *entropy, *top_lp;
    int32_t* top_idx;
    uint64_t row_stride;
    uint32_t rows, vocab, top_k;
    float scale;
};

template <int DT>
__device__ __forceinline__ float logit(const void* p, uint64_t i) {
    if constexpr (DT == GRAFT_F32) return ((const float*)p)[i];
    const uint16_t w = ((const uint16_t*)p)[i];
    return DT == GRAFT_F16 ? h2f(w) : bf2f(w);
}

template <int DT>
__global__ void __launch_bounds__(kThreads) logprobs_simple_kernel(const __grid_constant__ LpArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ float rv[kThreads];
    __shared__ double rs[kThreads], rt[kThreads];
    __shared__ int ri[kThreads];
    const int tid = threadIdx.x;
    const uint64_t row = blockIdx.x, base = row * a.row_stride;
    bool nan = false;
    float m = -INFINITY;
    for (uint32_t i = tid; i < a.vocab; i += kThreads) {
        const float z = logit<DT>(a.logits, base + i) * a.scale;
        nan |= !(z < INFINITY);
        m = fmaxf(m, z);
    }
    rv[tid] = m;
    nan = __syncthreads_or(nan);
    for (int s = kThreads / 2; s; s >>= 1) {
        if (tid < s) rv[tid] = fmaxf(rv[tid], rv[tid + s]);
        __syncthreads();
    }
    m = rv[0];
    __syncthreads();
    double L = 0, E = 0;   // sums of exp(z - m) and of it times (z - m)
    for (uint32_t i = tid; i < a.vocab; i += kThreads) {
        const float z = logit<DT>(a.logits, base + i) * a.scale;
        if (z > -INFINITY) {
            const float d = z - m, e = expf(d);
            L += e;
            E += (double)e * d;
        }
    }
    rs[tid] = L, rt[tid] = E;
    __syncthreads();
    for (int s = kThreads / 2; s; s >>= 1) {
        if (tid < s) rs[tid] += rs[tid + s], rt[tid] += rt[tid + s];
        __syncthreads();
    }
    L = rs[0], E = rt[0];
    const bool none = m == -INFINITY;
    const float lse = nan ? NAN : none ? 0.f : m + (float)log(L);
    if (tid == 0) {
        if (a.logprob) {
            const int t = a.targets[row];
            a.logprob[row] = (uint32_t)t < a.vocab
                                 ? logit<DT>(a.logits, base + t) * a.scale - lse : NAN;
        }
        if (a.entropy) a.entropy[row] = nan ? NAN : none ? 0.f : (float)(log(L) - E / L);
    }
    float pv = INFINITY;   // the alternative before: only what comes after it counts
    int pi = -1;
    for (uint32_t k = 0; k < a.top_k; ++k) {
        float bv = -INFINITY;
        int bi = -1;
        for (uint32_t i = tid; i < a.vocab; i += kThreads) {
            const float z = logit<DT>(a.logits, base + i);
            if (z > bv && (z < pv || (z == pv && (int)i > pi))) bv = z, bi = i;
        }
        rv[tid] = bv, ri[tid] = bi;
        __syncthreads();
        for (int s = kThreads / 2; s; s >>= 1) {
            if (tid < s) {
                const float v = rv[tid + s];
                const int i = ri[tid + s];
                if (i >= 0 && (v > rv[tid] || (v == rv[tid] && i < ri[tid]) || ri[tid] < 0))
                    rv[tid] = v, ri[tid] = i;
            }
            __syncthreads();
        }
        pv = rv[0], pi = ri[0];
        if (tid == 0) {
            a.top_idx[row * a.top_k + k] = pi;
            a.top_lp[row * a.top_k + k] = pi < 0 ? -INFINITY : pv * a.scale - lse;
        }
        __syncthreads();
        if (pi < 0) pi = 0x7FFFFFFF;
    }
}

int check_logprobs(const GraftLogprobParams* P) {
    clear_error();
    GRAFT_REQUIRE(P, "params pointer is null");
    GRAFT_REQUIRE(P->vocab >= 1 && P->vocab <= 0x7FFFFFFFu, "vocab %u out of range", P->vocab);
    GRAFT_REQUIRE(P->rows <= 0x7FFFFFFFu, "rows %u out of range", P->rows);
    GRAFT_REQUIRE(P->top_k <= 32, "top_k must be at most 32, not %u", P->top_k);
    GRAFT_REQUIRE(P->dtype <= GRAFT_F32, "unknown element type %u", P->dtype);
    GRAFT_REQUIRE(P->row_stride >= P->vocab || P->rows <= 1, "row_stride is below vocab");
    GRAFT_REQUIRE(std::isfinite(P->scale) && P->scale > 0.f, "scale must be positive and finite");
    return GRAFT_OK;
}

}  // namespace

extern "C" size_t graft_logprobs_workspace(const GraftLogprobParams* P) {
    return check_logprobs(P) ? 0 : 256;
}

extern "C" int graft_logprobs_init(void* ws, size_t ws_bytes, graft_stream_t stream) {
    clear_error();
    GRAFT_REQUIRE(ws && aligned(ws, 256), "the workspace must be 256-byte aligned");
    GRAFT_CUDA(cudaMemsetAsync(ws, 0, ws_bytes, stream));
    return GRAFT_OK;
}

extern "C" int graft_logprobs(const void* logits, const int32_t* targets, float* logprob,
                              float* entropy, float* top_logprob, int32_t* top_index,
                              const GraftLogprobParams* P, void* ws, size_t ws_bytes,
                              graft_stream_t stream) {
    int rc;
    if ((rc = check_logprobs(P))) return rc;
    const size_t need = graft_logprobs_workspace(P);
    GRAFT_REQUIRE(ws && aligned(ws, 256) && ws_bytes >= need,
                  "the workspace must be 256-byte aligned and hold %zu bytes", need);
    if (P->rows == 0) return GRAFT_OK;
    GRAFT_REQUIRE(logits && aligned(logits, P->dtype == GRAFT_F32 ? 4 : 2),
                  "logits must be a buffer aligned to its element type");
    GRAFT_REQUIRE(!logprob == !targets, "targets and logprob go together");
    GRAFT_REQUIRE(P->top_k == 0 || (top_logprob && top_index),
                  "top_logprob and top_index must be given for top_k %u", P->top_k);
    LpArgs a = {logits, targets, logprob, entropy, top_logprob, top_index, P->row_stride, P->rows,
                P->vocab, P->top_k, P->scale};
    void (*kern)(const LpArgs) = P->dtype == GRAFT_F16    ? logprobs_simple_kernel<GRAFT_F16>
                                 : P->dtype == GRAFT_BF16 ? logprobs_simple_kernel<GRAFT_BF16>
                                                          : logprobs_simple_kernel<GRAFT_F32>;
    return launch_pdl("logprobs", kern, dim3(P->rows), kThreads, 0, stream, a);
}
