// rope.cu -- rotary positions of queries and keys.
//
//   pair i of a head turns by p f_i:  (x, y) -> (x c - y s, y c + x s)
//
// Every element is read and written once: HBM bounds long calls, launch and load latency
// short ones.  A thread takes one unit (16 elements, 8 pairs) of several heads of a token,
// so that the 8 sines and cosines, which cost as much as turning the unit for ten heads, are
// computed once for them.
//
// Measured: 7687 tokens of 40 heads of 128 in bf16 27.9 us, 5.6 TB/s; 16 tokens 2.2 us.
#include "rope.cuh"

#include <algorithm>
#include <cmath>

using namespace graft;
using namespace graft::dev;

namespace {

struct RopeCall {
    const void* x;
    void* y;
    const int32_t* positions;
    uint64_t x_tok, x_head, y_tok, y_head;
    RopeArgs r;
    uint32_t tokens, heads, units;   // units of a head
    uint32_t groups;                 // threads a (token, unit); thread g takes heads g, g + groups, ..
    int copy;                        // out is another buffer: what is not turned is copied
};

constexpr int kRopeThreads = 256, kRopeHeads = 8;   // heads of a thread at most

template <int DT>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const __grid_constant__ RopeCall a) {
    pdl_wait();
    pdl_launch_dependents();
    const uint64_t at = (uint64_t)blockIdx.x * kRopeThreads + threadIdx.x;
    const uint32_t row = a.groups * a.units;
    const uint32_t t = (uint32_t)(at / row), in = (uint32_t)(at - (uint64_t)t * row);
    if (t >= a.tokens) return;
    const uint32_t g = in / a.units, k = in - g * a.units;
    const bool turned = (int)k < a.r.pairs;
    if (!turned && !a.copy) return;
    float c[8], s[8];
    if (turned) unit_turns<DT != GRAFT_F32>(a.r, k, a.positions[t], c, s);
    const uint64_t e0 = unit_chunk(a.r, k, 0) * 8, e1 = unit_chunk(a.r, k, 1) * 8;
    constexpr int UN = DT == GRAFT_F32 ? 2 : 4;
    for (uint32_t h0 = g; h0 < a.heads; h0 += UN * a.groups) {
        Raw<DT> p[UN], q[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u)
            if (h0 + u * a.groups < a.heads) {
                const uint64_t from = t * a.x_tok + (h0 + u * a.groups) * a.x_head;
                p[u] = load_own<DT>(a.x, from + e0), q[u] = load_own<DT>(a.x, from + e1);
            }
#pragma unroll
        for (int u = 0; u < UN; ++u)
            if (h0 + u * a.groups < a.heads) {
                const uint64_t to = t * a.y_tok + (h0 + u * a.groups) * a.y_head;
                if (turned) {
                    float x[8], y[8];
                    to_floats<DT>(p[u], x), to_floats<DT>(q[u], y);
                    turn_unit(a.r.half, c, s, x, y);
                    p[u] = from_floats<DT>(x), q[u] = from_floats<DT>(y);
                }
                store_raw<DT>(a.y, to + e0, p[u]), store_raw<DT>(a.y, to + e1, q[u]);
            }
    }
}

__global__ void rope_init_kernel(uint64_t* turns, const double* freqs, const GraftRopeParams P) {
    const int i = threadIdx.x;
    if (i >= (int)P.dims / 2) return;
    const double n = P.dims, pi = 3.14159265358979323846;
    double f;
    if (freqs) {
        f = freqs[i];
    } else {
        f = pow(P.base, -2.0 * i / n);
        if (P.scaling == GRAFT_ROPE_LINEAR) {
            f /= P.factor;
        } else if (P.scaling == GRAFT_ROPE_YARN) {
            const double per = n / (2 * log(P.base));
            const double lo = fmax(per * log(P.orig_len / (2 * pi * P.high)), 0.0);
            const double hi = fmin(per * log(P.orig_len / (2 * pi * P.low)), n - 1.0);
            const double r = fmin(fmax((i - lo) / fmax(hi - lo, 1e-3), 0.0), 1.0);
            f = f * (1 - r) + f / P.factor * r;
        } else if (P.scaling == GRAFT_ROPE_BANDS) {
            const double t = P.orig_len * f / (2 * pi);
            const double s = fmin(fmax((t - P.low) / (P.high - P.low), 0.0), 1.0);
            f = f * s + f / P.factor * (1 - s);
        }
    }
    // whole turns do not count; 2^64 itself is none
    double t = f / (2 * pi);
    t -= floor(t);
    turns[i] = t >= 1.0 ? 0 : (uint64_t)(t * 18446744073709551616.0);
}

template <int DT>
int launch_rope(const RopeCall& a, uint64_t threads, cudaStream_t st) {
    return launch_pdl("rope", rope_kernel<DT>, dim3((unsigned)((threads + kRopeThreads - 1) / kRopeThreads)),
                      kRopeThreads, 0, st, a);
}

}  // namespace

namespace graft {

int check_rope(const GraftRope* r, uint32_t head_dim) {
    GRAFT_REQUIRE(r, "rope is null");
    GRAFT_REQUIRE(r->turns && aligned(r->turns, 16), "rope: turns must be a 16-byte aligned buffer");
    GRAFT_REQUIRE(r->dims >= 16 && r->dims % 16 == 0 && r->dims <= head_dim,
                  "rope: dims must be a multiple of 16 up to head_dim %u, not %u", head_dim, r->dims);
    GRAFT_REQUIRE(r->layout <= GRAFT_ROPE_INTERLEAVED, "rope: unknown layout %u", r->layout);
    GRAFT_REQUIRE(std::isfinite(r->amplitude), "rope: amplitude must be finite");
    return GRAFT_OK;
}

RopeArgs rope_args(const GraftRope* r) {
    return RopeArgs{r->turns, r->amplitude, r->inverse ? -r->amplitude : r->amplitude,
                    (int)r->dims / 16, r->layout == GRAFT_ROPE_HALF};
}

int check_rope_rows(const GraftHeads* x, const GraftHeads* y, uint32_t heads) {
    int rc;
    GRAFT_REQUIRE(x && y, "x or out is null");
    if (heads == 0) return GRAFT_OK;   // (nothing: an empty buffer may have no address)
    if ((rc = kv_check_heads("x", x, 0)) || (rc = kv_check_heads("out", y, 0))) return rc;
    GRAFT_REQUIRE(heads <= 32767, "heads %u out of range", heads);
    GRAFT_REQUIRE(x->dtype == y->dtype && x->tokens == y->tokens,
                  "x and out must have the same type and number of tokens");
    GRAFT_REQUIRE((y->tokens <= 1 || y->token_stride) && (heads <= 1 || y->head_stride),
                  "the rows of out must not share memory");
    GRAFT_REQUIRE(x->data != y->data || y->tokens == 0 ||
                      (x->token_stride == y->token_stride && x->head_stride == y->head_stride),
                  "x and out must be the same rows or share no memory");
    return GRAFT_OK;
}

}  // namespace graft

extern "C" int graft_rope_init(uint64_t* turns, const double* freqs, const GraftRopeParams* P,
                               graft_stream_t stream) {
    clear_error();
    GRAFT_REQUIRE(P, "params pointer is null");
    GRAFT_REQUIRE(turns && aligned(turns, 16), "turns must be a 16-byte aligned buffer");
    GRAFT_REQUIRE(aligned(freqs, 8), "freqs must be 8-byte aligned");
    GRAFT_REQUIRE(P->dims >= 16 && P->dims % 16 == 0 && P->dims <= 256,
                  "dims must be a multiple of 16 up to 256, not %u", P->dims);
    if (!freqs) {
        GRAFT_REQUIRE(P->scaling <= GRAFT_ROPE_BANDS, "unknown scaling %u", P->scaling);
        GRAFT_REQUIRE(P->base > 0 && std::isfinite(P->base), "base must be positive and finite");
        GRAFT_REQUIRE(P->scaling == GRAFT_ROPE_PLAIN || (P->factor > 0 && std::isfinite(P->factor)),
                      "factor must be positive and finite");
        GRAFT_REQUIRE(P->scaling < GRAFT_ROPE_YARN ||
                          (P->orig_len > 0 && std::isfinite(P->orig_len) && P->low > 0 &&
                           P->low < P->high && std::isfinite(P->high)),
                      "orig_len must be positive and 0 < low < high");
        GRAFT_REQUIRE(P->scaling != GRAFT_ROPE_YARN || P->base != 1.0, "base must not be 1");
    }
    rope_init_kernel<<<1, 128, 0, stream>>>(turns, freqs, *P);
    return check_launch("rope_init");
}

extern "C" int graft_rope(const GraftHeads* x, const GraftHeads* out, uint32_t heads, uint32_t head_dim,
                          const int32_t* positions, const GraftRope* rope, graft_stream_t stream) {
    clear_error();
    int rc;
    if ((rc = check_rope_rows(x, out, heads))) return rc;
    GRAFT_REQUIRE(head_dim >= 16 && head_dim <= 256 && head_dim % 16 == 0,
                  "head_dim must be a multiple of 16 up to 256, not %u", head_dim);
    if ((rc = check_rope(rope, head_dim))) return rc;
    if (x->tokens == 0 || heads == 0) return GRAFT_OK;
    GRAFT_REQUIRE(positions && aligned(positions, 4), "positions must be a 4-byte aligned buffer");
    DeviceInfo di;
    if ((rc = current_device_info(&di))) return rc;
    RopeCall a = {};
    a.x = x->data, a.y = out->data, a.positions = positions;
    a.x_tok = x->token_stride, a.x_head = x->head_stride;
    a.y_tok = out->token_stride, a.y_head = out->head_stride;
    a.r = rope_args(rope);
    a.tokens = x->tokens, a.heads = heads, a.copy = x->data != out->data;
    a.units = head_dim / 16;
    // as many heads a thread as leave every SM four CTAs
    const uint64_t all = (uint64_t)a.tokens * a.units * heads;
    const uint64_t per = std::max<uint64_t>(1, std::min<uint64_t>(kRopeHeads, all / ((uint64_t)di.sm_count * 4 * kRopeThreads)));
    a.groups = (uint32_t)((heads + per - 1) / per);
    const uint64_t threads = (uint64_t)a.tokens * a.groups * a.units;
    GRAFT_REQUIRE(threads < (1ull << 38), "too many rows in one call");
    return x->dtype == GRAFT_F16    ? launch_rope<GRAFT_F16>(a, threads, stream)
           : x->dtype == GRAFT_BF16 ? launch_rope<GRAFT_BF16>(a, threads, stream)
                                    : launch_rope<GRAFT_F32>(a, threads, stream);
}
